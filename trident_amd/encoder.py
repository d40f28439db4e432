"""The operators of the encoder that makes and trains the vectors an index holds.

  embedding, embedding_grad            rows of a table for token ids, scaled; the table's gradient
  layer_norm, layer_norm_forward / _grad
  AdamW                                one launch per step for up to 88 tensors, states in 32 or 8 bits
  quantize_fp8, fp8_matmul, fp8_linear products in 8-bit floating point, one scale per row and 128 columns

``embedding`` and ``layer_norm`` take part in autograd; the ``*_forward`` / ``*_grad`` functions are the
bare passes; the 8-bit products have no gradient and refuse operands that require one.  Tensors with a
forward-mode tangent are refused.  Tensors are float32, float16 or bfloat16 on one GPU; sums, statistics
and states are float32 and every result is rounded once.  Each call runs on the current stream of its
tensors' device, with the library's workspace of that stream (``trident_amd.ext.workspace``), or, while a
graph is captured there, with scratch of the graph's own; results are the same bits every time.  Wrong
arguments raise ``TridentError``.

The reference has no counterpart: its vectors come from data sets.  The kernels are in libtrident_hip.so
(include/trident_hip.h); there is no fallback.
"""
from typing import Iterable, List, NamedTuple, Optional, Sequence, Tuple

import ctypes

import numpy as np
import torch
import torch.autograd.forward_ad as _forward_ad

from . import _lib, ext
from .ext import _need

_DTYPES = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}
_ID_TYPES = {torch.int32: 0, torch.int64: 1}
STATE_BLOCK = 256  # elements of an 8-bit state that share a scale

# A call on one query takes a few microseconds on the GPU, so the path to the library is kept short: the
# conditions are plain expressions, and messages are only made for a call that is refused.
_raw_stream, _current_device = ext._raw_stream, ext._current_device
_get_device, _data_ptr, _is_contiguous = torch.Tensor.get_device, torch.Tensor.data_ptr, torch.Tensor.is_contiguous
_increment_version = torch.autograd.graph.increment_version
_fns = {}


def _refuse(message: str) -> None:
    raise _lib.TridentError(message)


def _dtype(name: str, t: torch.Tensor) -> int:
    code = _DTYPES.get(t.dtype)
    if code is None:
        _refuse(f"{name} must be float32, float16 or bfloat16, got {t.dtype}")
    return code


def _gpu(name: str, t: torch.Tensor) -> int:
    """The index of the GPU that holds ``t``."""
    index = t.get_device()
    if index < 0:
        _refuse(f"{name} must be a device tensor, got one on {t.device}")
    return index


def _same(index: int, name: str, t: Optional[torch.Tensor]) -> None:
    if t is not None and t.get_device() != index:
        _refuse(f"{name} must be on cuda:{index}, got {t.device}")


def _rows(t: torch.Tensor) -> Tuple[torch.Tensor, int]:
    """(t, or a copy, with the elements of its last dimension next to each other and one pitch between
    its rows; that pitch)."""
    D = t.shape[-1]
    if not t.is_contiguous():
        if t.dim() != 2:
            t = t.reshape(-1, D)
        if (t.stride(1) != 1 and D != 1) or t.stride(0) < D:
            t = t.contiguous()
        elif t.shape[0] > 1:
            return t, t.stride(0)
    return t, max(D, 1)


def _no_tangents(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses dual tensors: the library computes values, and their tangents would be lost.  Called where
    a level of forward differentiation is open, ``_forward_ad._current_level >= 0``."""
    for t in tensors:
        if t is not None and _forward_ad.unpack_dual(t).tangent is not None:
            _refuse(f"{name} has no forward-mode derivative: an operand has a tangent")


def _constant(name: str, *tensors: Optional[torch.Tensor]) -> None:
    """Refuses operands whose gradient the caller could be waiting for: the products have none."""
    for t in tensors:
        if t is not None and t.requires_grad and torch.is_grad_enabled():
            _refuse(f"{name} has no gradient: pass detached tensors, or call it under torch.no_grad()")
    if _forward_ad._current_level >= 0:
        _no_tangents(name, *tensors)


def _fn(name: str):
    fn = _fns.get(name)
    if fn is None:
        fn = _fns[name] = getattr(_lib.lib(), name)
    return fn


def _call(index: int, name: str, *args) -> None:
    if index == _current_device():
        rc = _fn(name)(*args, _raw_stream(index))
    else:
        with torch.cuda.device(index):
            rc = _fn(name)(*args, _raw_stream(index))
    if rc:
        _lib.check(rc, name)


def _call_ws(device: torch.device, index: int, name: str, nbytes: int, *args) -> None:
    """_call with scratch of at least ``nbytes`` as the last two arguments, or, for none, without: this
    stream's workspace, or, under capture, memory of the graph's own (see ext._scratch)."""
    if nbytes == 0:
        return _call(index, name, *args, None, 0)
    slot = ext._ws_cache.get((device, _raw_stream(index)))
    if slot is None:
        slot = ext._workspace_slot(device, torch.cuda.current_stream(device))
    with slot.lock:
        ws = slot.buf
        if ws is None or ws.numel() < nbytes or index != _current_device() or ext._current_capturing():
            ws = ext._scratch(slot, device, nbytes, torch.cuda.current_stream(device))
        _call(index, name, *args, ws.data_ptr(), ws.numel())


# ---------------------------------------------------------------------------------------------
# embedding


def _ids(index: int, ids: torch.Tensor) -> Tuple[torch.Tensor, int]:
    wide = _ID_TYPES.get(ids.dtype)
    if wide is None:
        _refuse(f"ids must be int64 or int32, got {ids.dtype}")
    _same(index, "ids", ids)
    return (ids if ids.is_contiguous() else ids.contiguous()), wide


def _embed(ids, weight, scale):
    code, wide, index = _DTYPES.get(weight.dtype), _ID_TYPES.get(ids.dtype), weight.get_device()
    if code is None or wide is None or index < 0 or ids.get_device() != index or weight.dim() != 2 or \
            weight.numel() == 0:
        if weight.dim() != 2 or weight.numel() == 0:
            _refuse(f"weight must be [V, D], got {tuple(weight.shape)}")
        _dtype("weight", weight)
        _ids(_gpu("weight", weight), ids)
    V, D = weight.shape
    w, ld = (weight, D) if weight.is_contiguous() else _rows(weight)
    if not ids.is_contiguous():
        ids = ids.contiguous()
    out = weight.new_empty((*ids.shape, D))
    _call(index, "trident_embedding", w.data_ptr(), code, V, D, ld, ids.data_ptr(), wide, ids.numel(), scale,
          out.data_ptr(), D)
    return out


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, ids, weight, scale, padding_idx):
        ctx.save_for_backward(ids)
        ctx.rows, ctx.scale, ctx.padding_idx = weight.shape[0], scale, padding_idx
        return _embed(ids, weight, scale)

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        (ids,) = ctx.saved_tensors
        return None, embedding_grad(grad, ids, ctx.rows, ctx.scale, ctx.padding_idx), None, None


def embedding(ids: torch.Tensor, weight: torch.Tensor, scale: float = 1.0,
              padding_idx: Optional[int] = None) -> torch.Tensor:
    """``scale * weight[ids]``, shape ``[*ids.shape, D]`` in the table's type.

    A negative id is an empty slot of a padded batch and gives zeros; an id past the table gives NaN
    (the ids stay on the device, so no call can refuse them).  Neither has a gradient, nor has
    ``padding_idx``, whose row is looked up like any other.
    """
    if padding_idx is not None and not 0 <= padding_idx < len(weight):
        _refuse(f"padding_idx={padding_idx} outside [0, {len(weight)})")
    if _forward_ad._current_level >= 0:
        _no_tangents("embedding", weight)
    if weight.requires_grad and torch.is_grad_enabled():
        return _Embedding.apply(ids, weight, scale, padding_idx)
    return _embed(ids, weight, scale)


def embedding_grad(grad: torch.Tensor, ids: torch.Tensor, num_rows: int, scale: float = 1.0,
                   padding_idx: Optional[int] = None, out: Optional[torch.Tensor] = None) -> torch.Tensor:
    """The table's gradient ``[num_rows, D]`` in the type of ``grad`` (``[*ids.shape, D]``): row v is
    ``scale`` times the sum of the gradients of the tokens with id v.  Equal calls give equal bits; the order
    of a sum, and so its last bits, may change with the other tokens.  ``out`` (rows of any pitch) is written
    whole."""
    code, index = _dtype("grad", grad), _gpu("grad", grad)
    if _forward_ad._current_level >= 0:
        _no_tangents("embedding_grad", grad)
    if grad.dim() < 1 or grad.shape[:-1] != ids.shape or grad.shape[-1] == 0:
        _refuse(f"grad must be [*ids.shape, D], got {tuple(grad.shape)} for ids {tuple(ids.shape)}")
    if num_rows < 1:
        _refuse(f"num_rows must be positive, got {num_rows}")
    if padding_idx is not None and not 0 <= padding_idx < num_rows:
        _refuse(f"padding_idx={padding_idx} outside [0, {num_rows})")
    idc, wide = _ids(index, ids)
    n, D = idc.numel(), grad.shape[-1]
    g, ld = _rows(grad)
    ld_out = D
    if out is None:
        out = grad.new_empty((num_rows, D))
    else:
        _same(index, "out", out)
        if out.dtype != grad.dtype or tuple(out.shape) != (num_rows, D) or (out.stride(1) != 1 and D != 1) or \
                (out.stride(0) < D and num_rows > 1):
            _refuse(f"out must be [{num_rows}, {D}] {grad.dtype} with whole rows")
        if num_rows > 1:
            ld_out = out.stride(0)
    _call_ws(grad.device, index, "trident_embedding_grad", _fn("trident_embedding_grad_workspace_bytes")(n, num_rows, D),
             g.data_ptr(), code, ld, idc.data_ptr(), wide, n, num_rows, D, scale,
             -1 if padding_idx is None else padding_idx, out.data_ptr(), ld_out)
    return out


# ---------------------------------------------------------------------------------------------
# layer norm


def _affine(index, x, D, weight, bias) -> int:
    """The type code of weight and bias, which is x's or float32."""
    dtype = x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype
    for t in (weight, bias):
        if t is None:
            continue
        if t.shape != (D,) or not t.is_contiguous() or t.dtype is not dtype or t.get_device() != index:
            _refuse(f"weight and bias must be contiguous [{D}] of one type on cuda:{index}, got "
                    f"{[(tuple(t.shape), t.dtype, t.device) for t in (weight, bias) if t is not None]}")
    if dtype is not x.dtype and dtype is not torch.float32:
        _refuse(f"weight and bias must be {x.dtype} or float32, got {dtype}")
    return _DTYPES[dtype]


def _norm(x, weight, bias, eps, keep):
    code, index = _DTYPES.get(x.dtype), x.get_device()
    shape = x.shape
    D = shape[-1] if shape else 0
    if code is None or index < 0 or D == 0:
        _dtype("x", x)
        _gpu("x", x)
        _refuse(f"x must be [..., D], got {tuple(shape)}")
    wcode = code if weight is None and bias is None else _affine(index, x, D, weight, bias)
    if x.is_contiguous():
        xr, ld, y = x, D, torch.empty_like(x)
    else:
        (xr, ld), y = _rows(x), torch.empty_like(x, memory_format=torch.contiguous_format)
    mean = rstd = pmean = prstd = None
    if keep:
        mean = x.new_empty(shape[:-1], dtype=torch.float32)
        rstd = torch.empty_like(mean)
        pmean, prstd = mean.data_ptr(), rstd.data_ptr()
    _call(index, "trident_layer_norm", xr.data_ptr(), code, x.numel() // D, D, ld,
          None if weight is None else weight.data_ptr(), None if bias is None else bias.data_ptr(), wcode, eps,
          y.data_ptr(), D, pmean, prstd)
    return y, mean, rstd


class _LayerNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, eps):
        y, mean, rstd = _norm(x, weight, bias, eps, True)
        ctx.save_for_backward(x, weight, mean, rstd)
        ctx.bias_dtype = None if bias is None else bias.dtype
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, grad):
        x, weight, mean, rstd = ctx.saved_tensors
        dx, dw, db = _norm_grad(grad, x, weight, mean, rstd, ctx.needs_input_grad[1], ctx.needs_input_grad[2],
                                ctx.bias_dtype if weight is None else weight.dtype)
        return (dx if ctx.needs_input_grad[0] else None), dw, db, None


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5) -> torch.Tensor:
    """Layer norm over the last dimension of ``x``; ``weight`` and ``bias`` ([D], of x's type or
    float32) may be left out."""
    if _forward_ad._current_level >= 0:
        _no_tangents("layer_norm", x, weight, bias)
    if torch.is_grad_enabled() and (x.requires_grad or (weight is not None and weight.requires_grad) or
                                    (bias is not None and bias.requires_grad)):
        return _LayerNorm.apply(x, weight, bias, eps)
    return _norm(x, weight, bias, eps, False)[0]


def layer_norm_forward(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
                       eps: float = 1e-5) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(y, mean, rstd): layer norm and the rows' float32 statistics, which the backward pass takes."""
    if _forward_ad._current_level >= 0:
        _no_tangents("layer_norm_forward", x, weight, bias)
    return _norm(x, weight, bias, eps, True)


def layer_norm_grad(grad: torch.Tensor, x: torch.Tensor, weight: Optional[torch.Tensor], mean: torch.Tensor,
                    rstd: torch.Tensor):
    """(dx, dweight, dbias) from the gradient of y and what ``layer_norm_forward`` kept; the last two in
    the weight's type (x's without a weight, and then no dweight)."""
    return _norm_grad(grad, x, weight, mean, rstd, weight is not None, True, x.dtype if weight is None else weight.dtype)


def _norm_grad(grad, x, weight, mean, rstd, need_w, need_b, wdtype):
    if _forward_ad._current_level >= 0:
        _no_tangents("layer_norm_grad", grad, x, weight, mean, rstd)
    code, index = _DTYPES.get(x.dtype), x.get_device()
    shape, lead = x.shape, x.shape[:-1]
    D = shape[-1] if shape else 0
    if code is None or index < 0 or D == 0 or grad.shape != shape or grad.dtype is not x.dtype or \
            grad.get_device() != index:
        _dtype("x", x)
        _gpu("x", x)
        if D == 0:
            _refuse(f"x must be [..., D], got {tuple(shape)}")
        if grad.shape != shape or grad.dtype is not x.dtype:
            _refuse(f"grad must be {tuple(shape)} {x.dtype}, got {tuple(grad.shape)} {grad.dtype}")
        _same(index, "grad", grad)
    if mean.dtype is not torch.float32 or rstd.dtype is not torch.float32 or mean.shape != lead or \
            rstd.shape != lead or not mean.is_contiguous() or not rstd.is_contiguous() or \
            mean.get_device() != index or rstd.get_device() != index:
        _refuse(f"mean and rstd must be contiguous float32 {tuple(lead)} on cuda:{index}")
    if weight is not None:
        _affine(index, x, D, weight, None)
    wcode = code if wdtype is None else _DTYPES[wdtype]
    rows = x.numel() // D
    xr, ldx = (x, D) if x.is_contiguous() else _rows(x)
    gr, ldg = (grad, D) if grad.is_contiguous() else _rows(grad)
    dx = torch.empty_like(x, memory_format=torch.contiguous_format)
    dw = db = pdw = pdb = None
    if need_w:
        dw = torch.empty_like(weight)
        pdw = dw.data_ptr()
    if need_b:
        db = x.new_empty(D, dtype=wdtype) if weight is None else torch.empty_like(weight)
        pdb = db.data_ptr()
    _call_ws(x.device, index, "trident_layer_norm_grad", _fn("trident_layer_norm_grad_workspace_bytes")(rows, D),
             gr.data_ptr(), ldg, xr.data_ptr(), ldx, code, rows, D, None if weight is None else weight.data_ptr(),
             wcode, mean.data_ptr(), rstd.data_ptr(), dx.data_ptr(), D, pdw, pdb)
    return dx, dw, db


# ---------------------------------------------------------------------------------------------
# AdamW

_TABLE = np.dtype([("param", "u8"), ("grad", "u8"), ("numel", "i8"), ("offset", "i8"), ("dtype", "i4"),
                   ("grad_dtype", "i4")])  # TridentAdamTensor


class AdamW:
    """AdamW (decoupled weight decay) over a list of tensors of float32, float16 or bfloat16.

    A class of its own, not a ``torch.optim.Optimizer``: schedulers and gradient scalers that ask for one do
    not take it; set ``lr`` and pass ``grad_scale`` instead.

    ``step()`` updates the parameters in place from their ``.grad`` (or from a list of gradients, each of
    any of the three types); a parameter without one is left alone, though the step count, which is the
    optimizer's, goes on for all.  ``grad_scale`` multiplies the gradients (one over a loss scale).  ``lr``,
    ``weight_decay`` and ``step_count`` may be set between steps; groups with other settings are other
    optimizers.

    The moments are float32 (``state_bits=32``) or 8-bit codes with a float32 scale for every 256
    (``state_bits=8``: 2.03 bytes a parameter instead of 8); the arithmetic is float32 either way.  They
    lie in flat buffers ``exp_avg`` and ``exp_avg_sq`` (with ``exp_avg_scale`` and ``exp_avg_sq_scale``),
    tensor i's from ``offsets[i]``, a multiple of 256, zeros up to the next tensor's.  A gradient that is
    not finite shows in its parameter and state; in 8 bits in the state of its block of 256.

    8-bit codes are the nearest ones in the first 2 / (1 - betas[0]) steps.  After them each is one of the two
    around its value, chosen by a hash (of place, step and the block's largest moments) so that the moment is
    right in the mean: one that changes by less than a code a step still falls or grows as it should.

    A step captured in a graph takes the learning rate and the step count of its capture at every replay.
    """

    def __init__(self, params: Iterable[torch.Tensor], lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999),
                 eps: float = 1e-8, weight_decay: float = 1e-2, state_bits: int = 32):
        self.params: List[torch.Tensor] = list(params)
        _need(len(self.params) > 0, "AdamW needs at least one parameter")
        _need(state_bits in (8, 32), f"state_bits must be 8 or 32, got {state_bits}")
        _need(0.0 <= betas[0] < 1.0 and 0.0 <= betas[1] < 1.0, f"betas must lie in [0, 1), got {betas}")
        _need(lr >= 0.0 and eps >= 0.0 and weight_decay >= 0.0, "lr, eps and weight_decay must not be negative")
        _need(len({id(p) for p in self.params}) == len(self.params), "a parameter is listed twice")
        self.device, self._index = self.params[0].device, _gpu("parameter 0", self.params[0])
        self.lr, self.betas, self.eps, self.weight_decay = float(lr), tuple(betas), float(eps), float(weight_decay)
        self.state_bits, self.step_count = state_bits, 0
        self.offsets, total = [], 0
        for i, p in enumerate(self.params):
            _dtype(f"parameter {i}", p)
            _same(self._index, f"parameter {i}", p)
            _need(p.is_contiguous(), f"parameter {i} must be contiguous")
            self.offsets.append(total)
            total += -(-p.numel() // STATE_BLOCK) * STATE_BLOCK
        self._apart = None  # the last step's parameters, by address and type, which share no memory
        self._need_apart(self.params, list(map(_data_ptr, self.params)))
        self._shapes = [p.shape for p in self.params]
        self._table = np.zeros(len(self.params), _TABLE)
        self._table["numel"] = [p.numel() for p in self.params]
        self._table["offset"] = self.offsets
        self._table_at = self._table.ctypes.data
        self._kinds = None  # the types of parameters and gradients that the table names
        kind = (torch.float32, torch.float32) if state_bits == 32 else (torch.int8, torch.uint8)
        moments = [torch.zeros(total, dtype=k, device=self.device) for k in kind]
        scales = [torch.zeros(total // STATE_BLOCK, device=self.device) if state_bits == 8 else None for _ in kind]
        self._buffers = (*moments, *scales)
        self._state = _lib.TridentAdamState(*map(ext._ptr, self._buffers), total, state_bits)

    @staticmethod
    def _need_apart(params, addresses) -> None:
        """A step reads and writes each element once, by workgroups that know nothing of each other."""
        spans = sorted((a, a + p.numel() * p.element_size()) for p, a in zip(params, addresses) if p.numel())
        if not all(a[1] <= b[0] for a, b in zip(spans, spans[1:])):
            _refuse("parameters share memory")

    def zero_grad(self) -> None:
        for p in self.params:
            p.grad = None

    def step(self, grads: Optional[Sequence[Optional[torch.Tensor]]] = None, grad_scale: float = 1.0) -> None:
        grads = [p.grad for p in self.params] if grads is None else list(grads)
        if len(grads) != len(self.params):
            _refuse(f"{len(self.params)} gradients are needed, got {len(grads)}")
        params, shapes, table = self.params, self._shapes, self._table
        try:
            devices = set(map(_get_device, grads))
        except TypeError:  # one is None
            at = [i for i, g in enumerate(grads) if g is not None]
            params, shapes, grads = [params[i] for i in at], [shapes[i] for i in at], [grads[i] for i in at]
            table = table[at]
            devices = set(map(_get_device, grads))
        devices.update(map(_get_device, params))
        if [g.shape for g in grads] != shapes or not devices <= {self._index}:
            _refuse(f"gradients must be on {self.device} and of their parameters' shapes "
                    f"{[tuple(s) for s in shapes]}, got {[(tuple(g.shape), g.device) for g in grads]}")
        if [p.shape for p in params] != shapes or not all(map(_is_contiguous, params)):
            _refuse("a parameter is no longer the contiguous tensor it was")
        try:
            if not all(map(_is_contiguous, grads)):
                grads = [g.detach().contiguous() for g in grads]
            table["grad"] = [*map(_data_ptr, grads)]
        except RuntimeError as e:  # sparse
            _refuse(f"gradients must be dense: {e}")
        kinds = [p.dtype for p in params], [g.dtype for g in grads]
        whole = table is self._table
        if not whole or kinds != self._kinds:  # else the table has them
            try:
                codes = [[_DTYPES[t] for t in of] for of in kinds]
            except KeyError as e:
                _refuse(f"parameters and gradients must be float32, float16 or bfloat16, got {e}")
            table["dtype"], table["grad_dtype"] = codes
            if whole:
                self._kinds = kinds
        addresses = [*map(_data_ptr, params)]
        if (addresses, kinds[0]) != self._apart:
            self._need_apart(params, addresses)
            self._apart = addresses, kinds[0]
        table["param"] = addresses
        h = _lib.TridentAdamParams(self.lr, self.betas[0], self.betas[1], self.eps, self.weight_decay, grad_scale,
                                   self.step_count + 1)
        _call(self._index, "trident_adamw", self._table_at if whole else table.ctypes.data, len(params),
              ctypes.byref(self._state), ctypes.byref(h))
        self.step_count += 1
        _increment_version(params)

    # the states' buffers: to be read or changed in place (the library holds their addresses)
    exp_avg = property(lambda self: self._buffers[0])
    exp_avg_sq = property(lambda self: self._buffers[1])
    exp_avg_scale = property(lambda self: self._buffers[2])
    exp_avg_sq_scale = property(lambda self: self._buffers[3])

    def state_values(self) -> Tuple[torch.Tensor, torch.Tensor]:
        """The moments as flat float32 tensors: the buffers themselves, or what the 8-bit codes stand for."""
        if self.state_bits == 32:
            return self.exp_avg, self.exp_avg_sq
        m, v = torch.empty((2, self.exp_avg.numel()), device=self.device)
        _call(self._index, "trident_adamw_state_values", ctypes.byref(self._state), m.data_ptr(), v.data_ptr())
        return m, v

    def load_state(self, step_count: int, exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor,
                   exp_avg_scale: Optional[torch.Tensor] = None,
                   exp_avg_sq_scale: Optional[torch.Tensor] = None) -> None:
        """Copies flat states (as the attributes of the same names hold them) and the steps taken."""
        _need(step_count >= 0, f"step_count must not be negative, got {step_count}")
        given = dict(exp_avg=exp_avg, exp_avg_sq=exp_avg_sq, exp_avg_scale=exp_avg_scale,
                     exp_avg_sq_scale=exp_avg_sq_scale)
        for name, t in given.items():
            mine = getattr(self, name)
            _need((t is None) == (mine is None), f"{name} does not go with states of {self.state_bits} bits")
            _need(t is None or (t.dtype == mine.dtype and t.numel() == mine.numel()),
                  f"{name} must be {None if mine is None else (mine.numel(), mine.dtype)}")
        for name, t in given.items():
            if t is not None:
                getattr(self, name).copy_(t.reshape(-1))
        self.step_count = int(step_count)

    def state_dict(self) -> dict:
        names = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
        return dict(step_count=self.step_count, state_bits=self.state_bits, numels=self._table["numel"].tolist(),
                    **{n: getattr(self, n).clone() for n in names if getattr(self, n) is not None})

    def load_state_dict(self, state: dict) -> None:
        """Takes what ``state_dict`` gave, for tensors of the same sizes in the same order (``numels``; a state
        saved without them has to have the same length in all)."""
        _need(state.get("state_bits") == self.state_bits,
              f"the state has {state.get('state_bits')} bits, this optimizer {self.state_bits}")
        numels = self._table["numel"].tolist()
        _need(list(state.get("numels", numels)) == numels,
              f"the state is of tensors of {state.get('numels')} elements, the parameters have {numels}")
        self.load_state(state["step_count"], state["exp_avg"], state["exp_avg_sq"], state.get("exp_avg_scale"),
                        state.get("exp_avg_sq_scale"))


# ---------------------------------------------------------------------------------------------
# 8-bit floating point


class Fp8Blocks(NamedTuple):
    """A matrix [rows, K] as e4m3 codes with one scale ``2**(scales - 127)`` per row and 128 columns:
    ``codes`` [rows, 128 ceil(K / 128)] float8_e4m3fn (zeros past K), ``scales`` [rows, 4 ceil(K / 512)]
    uint8 (127 past the last block)."""
    codes: torch.Tensor
    scales: torch.Tensor
    K: int


def _fp8_pitches(K: int) -> Tuple[int, int]:
    return -(-K // 128) * 128, -(-K // 512) * 4


def _check_blocks(name: str, b: Fp8Blocks, index: int) -> int:
    if not isinstance(b, Fp8Blocks):
        _refuse(f"{name} must be Fp8Blocks (quantize_fp8)")
    codes, scales, K = b
    rows = codes.shape[0]
    if codes.dtype is not torch.float8_e4m3fn or scales.dtype is not torch.uint8 or K < 1 or \
            codes.shape != (rows, -(-K // 128) * 128) or scales.shape != (rows, -(-K // 512) * 4) or \
            not codes.is_contiguous() or not scales.is_contiguous():
        _refuse(f"{name} must hold contiguous float8_e4m3fn codes {(rows,) + _fp8_pitches(K)[:1]} and uint8 scales "
                f"{(rows,) + _fp8_pitches(K)[1:]} for K={K}, got {codes.dtype} {tuple(codes.shape)} and "
                f"{scales.dtype} {tuple(scales.shape)}")
    if codes.get_device() != index or scales.get_device() != index:
        _refuse(f"{name} must be on cuda:{index}")
    return rows


def quantize_fp8(x: torch.Tensor) -> Fp8Blocks:
    """``x`` [rows, K] in 8-bit floating point: each row's 128 columns share the least power of two under
    which their largest value is at most 448.  A value that is not finite becomes NaN.  No gradient: ``x``
    that requires one is refused under grad mode."""
    code, index = _dtype("x", x), _gpu("x", x)
    _constant("quantize_fp8", x)
    if x.dim() != 2 or x.shape[1] == 0:
        _refuse(f"x must be [rows, K], got {tuple(x.shape)}")
    rows, K = x.shape
    xr, ld = _rows(x)
    kp, sp = _fp8_pitches(K)
    codes, scales = x.new_empty((rows, kp), dtype=torch.float8_e4m3fn), x.new_empty((rows, sp), dtype=torch.uint8)
    _call(index, "trident_fp8_quantize", xr.data_ptr(), code, rows, K, ld, codes.data_ptr(), scales.data_ptr())
    return Fp8Blocks(codes, scales, K)


def _bias(bias, N, dtype, index) -> int:
    if bias is None:
        return _DTYPES[dtype]
    if bias.shape != (N,) or not bias.is_contiguous():
        _refuse(f"bias must be a contiguous [{N}]")
    if bias.dtype is not dtype and bias.dtype is not torch.float32:
        _refuse(f"bias must be {dtype} or float32, got {bias.dtype}")
    _same(index, "bias", bias)
    return _DTYPES[bias.dtype]


def fp8_matmul(a: Fp8Blocks, b: Fp8Blocks, bias: Optional[torch.Tensor] = None,
               out_dtype: torch.dtype = torch.bfloat16, fast_accum: bool = False) -> torch.Tensor:
    """``a @ b.T + bias``: [M, N] from [M, K] and [N, K], summed in float32.

    ``fast_accum`` takes the 8-bit matrix instruction, which is twice as fast and keeps 13 bits below the
    largest of each 8 products: the sums are off by up to about 5e-5 of their size, which a bfloat16
    result does not show.  No gradient: a bias that requires one is refused under grad mode."""
    if not isinstance(a, Fp8Blocks):
        _refuse("a must be Fp8Blocks (quantize_fp8)")
    index = _gpu("a", a.codes)
    M, N = _check_blocks("a", a, index), _check_blocks("b", b, index)
    if a.K != b.K:
        _refuse(f"a has {a.K} columns, b {b.K}")
    if out_dtype not in _DTYPES:
        _refuse(f"out_dtype must be float32, float16 or bfloat16, got {out_dtype}")
    bcode = _bias(bias, N, out_dtype, index)
    _constant("fp8_matmul", bias)
    out = a.codes.new_empty((M, N), dtype=out_dtype)
    _call(index, "trident_fp8_matmul", a.codes.data_ptr(), a.scales.data_ptr(), M, b.codes.data_ptr(),
          b.scales.data_ptr(), N, a.K, None if bias is None else bias.data_ptr(), bcode, out.data_ptr(),
          _DTYPES[out_dtype], max(N, 1), fast_accum)
    return out


def fp8_linear(x: torch.Tensor, weight: Fp8Blocks, bias: Optional[torch.Tensor] = None,
               fast_accum: bool = False) -> torch.Tensor:
    """``x @ weight.T + bias`` for ``x`` [..., K], quantised in the call, in x's type: the projection of a
    query or a corpus by a weight kept in 8 bits.  ``fast_accum``: see ``fp8_matmul``.  No gradient: ``x`` or
    a bias that requires one is refused under grad mode."""
    code, index = _DTYPES.get(x.dtype), x.get_device()
    if code is None or index < 0:
        _dtype("x", x)
        _gpu("x", x)
    N = _check_blocks("weight", weight, index)
    codes, scales, K = weight
    shape = x.shape
    if not shape or shape[-1] != K:
        _refuse(f"x must be [..., {K}], got {tuple(shape)}")
    M = x.numel() // K
    bcode, bptr = code, None
    if bias is not None:
        bcode, bptr = _bias(bias, N, x.dtype, index), bias.data_ptr()
    if x.requires_grad or (bias is not None and bias.requires_grad) or _forward_ad._current_level >= 0:
        _constant("fp8_linear", x, bias)
    xr, ld = (x, K) if x.is_contiguous() else _rows(x)
    out = x.new_empty((M, N) if len(shape) == 2 else (*shape[:-1], N))
    _call_ws(x.device, index, "trident_fp8_linear", _fn("trident_fp8_linear_workspace_bytes")(M, N, K), xr.data_ptr(),
             code, M, K, ld, codes.data_ptr(), scales.data_ptr(), N, bptr, bcode, out.data_ptr(), N or 1, fast_accum)
    return out
