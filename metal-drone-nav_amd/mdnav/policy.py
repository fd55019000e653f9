"""Operators of a policy network and its loss over torch tensors on the GPU:
the linear layer with bias, activation and residual (``linear``), the gated
feed-forward block (``gated_feed_forward``) and the clipped loss of a policy
over discrete choices (``clipped_loss``), all with gradients, and the
log-probabilities that acting stores for that loss (``log_prob``).

They go with ``sequence``, whose ``block_norm`` has the norms around such a
block, and follow its rules: device tensors as they are, on torch's current
stream; an argument that is a lazily negated view is to be resolved before (a
gradient that arrives as one is resolved here); torch is imported before the
library is first used.
"""
import ctypes
import struct

import torch
import torch.autograd.function

from .native import P, check
from .sequence import (_DTYPES, _address, _buffer, _device, _library, _like, _no_tangents, _number, _on, _shape, _stream,
                       _wide)

ACTIVATIONS = {"none": 0, "relu": 1, "tanh": 2, "sigmoid": 3, "silu": 4, "gelu": 5, "gelu_tanh": 6}


class _Matrix(ctypes.Structure):
    _fields_ = [("data", P), ("row", ctypes.c_int64)]


class _Dense(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_uint64)]
    _fields_ += [(n, ctypes.c_uint32) for n in ("in_", "out", "dtype", "activation", "gated")]
    _fields_ += [(n, _Matrix) for n in ("x", "w", "w_up", "residual", "y")]
    _fields_ += [("b", P), ("b_up", P)]


class _DenseGrad(ctypes.Structure):
    _fields_ = [(n, _Matrix) for n in ("d_y", "d_x", "d_w", "d_w_up")]
    _fields_ += [("d_b", P), ("d_b_up", P)]


class _Choices(ctypes.Structure):
    _fields_ = [("steps", ctypes.c_uint64)]
    _fields_ += [(n, ctypes.c_uint32) for n in ("heads", "choices", "dtype", "action_bytes")]
    _fields_ += [("logits", P), ("step", ctypes.c_int64), ("head", ctypes.c_int64), ("actions", P)]


class _ChoiceLoss(ctypes.Structure):
    _fields_ = [(n, P) for n in ("old_log_prob", "advantages", "ref_log_prob", "mask")]
    _fields_ += [(n, ctypes.c_double) for n in ("clip_low", "clip_high", "kl_coef", "entropy_coef")]
    _fields_ += [("loss", P), ("metrics", P)]


# The structs as packed bytes, made of plain numbers in one call each.
_DENSE = struct.Struct("=Q5I4x12q")
_DENSE_GRAD = struct.Struct("=10q")
assert _DENSE.size == ctypes.sizeof(_Dense) and _DENSE_GRAD.size == ctypes.sizeof(_DenseGrad)
_CHOICES = struct.Struct("=Q4I4q")
_CHOICE_LOSS = struct.Struct("=4q4d2q")
assert _CHOICES.size == ctypes.sizeof(_Choices) and _CHOICE_LOSS.size == ctypes.sizeof(_ChoiceLoss)
_NONE = (0, 0)


def _matrix(t):
    """The rows of `t`, [..., width], as an address and the elements from row to row; another layout is copied.
    The tensor is returned too: it holds the memory."""
    if t.is_contiguous():
        return t, (t.data_ptr(), t.shape[-1])
    t = _wide(t)
    row = None
    for size, stride in zip(reversed(t.shape[:-1]), reversed(t.stride()[:-1])):
        if size == 1:
            continue
        if row is None:
            row, joined = stride, size * stride
        elif stride == joined:
            joined *= size
        else:
            t = t.contiguous()
            return t, (t.data_ptr(), t.shape[-1])
    return t, (t.data_ptr(), t.shape[-1] if row is None else row)


class _Kept:
    """A call for its gradient: the structs with the addresses of what autograd saves, and none of the tensors.  (Checking
    them anew takes 15 of the 120 us that a small loss and its gradient do.)"""

    def __init__(self, call, saved):
        self.call = call if all([t is None or t.is_contiguous() for t in saved]) else None
        self.at = [None if t is None else (t.data_ptr(), t.shape) for t in saved]
        call.drop()

    def again(self, saved):
        """The call, if what was saved is as it was, or None: a hook or an assignment to .data may have changed it."""
        if self.call is None:
            return None
        for t, at in zip(saved, self.at):
            if t is not None and (t.data_ptr() != at[0] or t.shape != at[1] or not t.is_contiguous()):
                return None
        return self.call


class _DenseCall:
    """Checked arguments of one call of a linear layer or a gated block: the C struct and what it points to."""

    def __init__(self, names, x, w, w_up, b, b_up, residual, activation):
        self.device = _device(names, (x, w, w_up, b, b_up, residual))
        activation = "none" if activation is None else activation
        if activation not in ACTIVATIONS:
            raise ValueError("activation is one of %s, not %r" % (", ".join(ACTIVATIONS), activation))
        if x.dim() < 1:
            raise ValueError("x is [..., in]")
        if w.dim() != 2:
            raise ValueError("%s is [out, in]" % names[1])
        out, width = w.shape
        _shape("x", x, (*x.shape[:-1], width))
        if not 1 <= width <= 65536 or not 1 <= out <= 65536:
            raise ValueError("widths are 1..65536, not %d and %d" % (width, out))
        dtype = x.dtype
        if dtype not in _DTYPES:
            raise TypeError("x is %s: float32 or bfloat16 are taken" % dtype)
        self.shape = (*x.shape[:-1], out)
        for name, t, shape in zip(names[1:], (w, w_up, b, b_up, residual), (w.shape, w.shape, (out,), (out,), self.shape)):
            if t is None:
                continue
            _shape(name, t, shape)
            if t.dtype != dtype:
                raise TypeError("%s is %s and x %s: one type is taken" % (name, t.dtype, dtype))
        self.rows, self.gated, self.dtype = x.numel() // width, w_up is not None, dtype
        if self.rows > 0x7fffff00:
            raise ValueError("%d rows are too many" % self.rows)
        self.x, mx = _matrix(x)
        self.w, mw = _matrix(w)
        self.w_up, mu = (None, _NONE) if w_up is None else _matrix(w_up)
        self.residual, mr = (None, _NONE) if residual is None else _matrix(residual)
        self.b, self.b_up = (None if t is None else t.contiguous() for t in (b, b_up))
        self.c = _Dense.from_buffer_copy(_DENSE.pack(
            self.rows, width, out, _DTYPES[dtype], ACTIVATIONS[activation], self.gated, *mx, *mw, *mu, *mr, *_NONE,
            _address(self.b) or 0, _address(self.b_up) or 0))

    def forward(self):
        L = _library()
        y = torch.empty(self.shape, dtype=self.dtype, device=self.device)
        c = self.c
        c.y.data, c.y.row = y.data_ptr(), c.out
        size = ctypes.c_uint64()
        check(L.mdn_op_dense_forward_bytes(ctypes.byref(c), ctypes.byref(size)))
        work = _buffer(size.value, self.device)
        check(L.mdn_op_dense_forward(ctypes.byref(c), _address(work), size.value, _stream(self.device)))
        return y

    def drop(self):
        self.x = self.w = self.w_up = self.b = self.b_up = self.residual = None

    def backward(self, d_y, inputs, want):
        """(d_x, d_w, d_w_up, d_b, d_b_up), None where `want` is false"""
        L = _library()
        d_y, my = _matrix(d_y.resolve_neg())
        made = [_like(t) if wanted and t is not None else None for wanted, t in zip(want, inputs)]
        if self.rows == 0:
            return [None if t is None else t.zero_() for t in made]
        at = [(0 if t is None else t.data_ptr(), 0 if t is None else t.shape[-1]) for t in made]
        d = _DenseGrad.from_buffer_copy(_DENSE_GRAD.pack(*my, *at[0], *at[1], *at[2], at[3][0], at[4][0]))
        size = ctypes.c_uint64()
        check(L.mdn_op_dense_backward_bytes(ctypes.byref(self.c), ctypes.byref(d), ctypes.byref(size)))
        work = _buffer(size.value, self.device)
        check(L.mdn_op_dense_backward(ctypes.byref(self.c), ctypes.byref(d), _address(work), size.value,
                                      _stream(self.device)))
        return made


class _DenseFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, names, activation, x, w, w_up, b, b_up, residual):
        call = _DenseCall(names, x, w, w_up, b, b_up, residual, activation)
        y = _on(call.device, call.forward)
        saved = (x, w, w_up, b, b_up)
        ctx.names, ctx.activation, ctx.like, ctx.kept = names, activation, residual is not None, _Kept(call, saved)
        ctx.save_for_backward(*saved)
        return y

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_y):
        want = ctx.needs_input_grad
        d_residual = d_y if ctx.like and want[7] else None
        if not any(want[2:7]):
            return (*[None] * 7, d_residual)
        saved = ctx.saved_tensors
        call = ctx.kept.again(saved) or _DenseCall(ctx.names, *saved, None, ctx.activation)
        grads = _on(call.device, call.backward, d_y, saved, want[2:7])
        return (None, None, *grads, d_residual)


def _dense(names, activation, *args):
    _no_tangents(*args)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in args):
        return _DenseFunction.apply(names, activation, *args)
    call = _DenseCall(names, *args, activation)
    return _on(call.device, call.forward)


_LINEAR = ("x", "weight", "weight", "bias", "bias", "residual")
_GATED = ("x", "w_gate", "w_up", "b_gate", "b_up", "residual")


def _tensors(**args):
    for name, t in args.items():
        if not isinstance(t, torch.Tensor):
            raise TypeError("%s is no tensor" % name)


def linear(x, weight, bias=None, activation=None, residual=None):
    """residual + act(x weight^T + bias), rounded once.

    x: [..., in], weight: [out, in], bias: [out], residual: [..., out], all
    float32 or all bfloat16; widths up to 65,536.  activation: "none" (or
    None), "relu", "tanh", "sigmoid", "silu", "gelu" or "gelu_tanh".  Any
    leading strides go; operands whose rows are not whole, aligned 16-byte
    words are copied first.  Gradients reach every tensor argument; the
    activation's argument is made again for them and not kept, and its gradient
    enters the products that follow with the rows' type.
    """
    _tensors(x=x, weight=weight)
    return _dense(_LINEAR, activation, x, weight, None, bias, None, residual)


def gated_feed_forward(x, w_gate, w_up, b_gate=None, b_up=None, activation="silu"):
    """act(x w_gate^T + b_gate) * (x w_up^T + b_up), rounded once.

    x: [..., in], w_gate, w_up: [out, in], b_gate, b_up: [out]; types,
    activations, strides and gradients as in ``linear``.
    """
    _tensors(x=x, w_gate=w_gate, w_up=w_up)
    return _dense(_GATED, activation, x, w_gate, w_up, b_gate, b_up, None)


# ---------------------------------------------------------------- discrete choices
class _ChoiceCall:
    """Checked logits and actions: the C struct and what it points to."""

    def __init__(self, logits, actions, more=(), names=()):
        self.device = _device(("logits", "actions", *names), (logits, actions, *more))
        if logits.dim() < 2:
            raise ValueError("logits are [..., heads, choices]")
        heads, choices = logits.shape[-2:]
        self.shape = logits.shape[:-2]
        _shape("actions", actions, logits.shape[:-1])
        if heads < 1 or heads > 65536 or choices < 1 or choices >= 1 << 24:
            raise ValueError("heads are 1..65536 and choices 1..2^24 - 1, not %d and %d" % (heads, choices))
        if logits.dtype not in _DTYPES:
            raise TypeError("logits are %s: float32 or bfloat16 are taken" % logits.dtype)
        if actions.dtype not in (torch.int64, torch.int32):
            raise TypeError("actions are %s: int64 or int32 are taken" % actions.dtype)
        self.steps = logits.numel() // (heads * choices)
        if logits.is_contiguous():
            rows, strides = logits, (heads * choices, choices)
        else:
            rows = _wide(logits)
            try:
                rows = rows.view(self.steps, heads, choices)
            except RuntimeError:
                rows = rows.contiguous().view(self.steps, heads, choices)
            strides = rows.stride()[:2]
        self.logits, self.actions = rows, actions.contiguous()
        self.c = _Choices.from_buffer_copy(_CHOICES.pack(
            self.steps, heads, choices, _DTYPES[logits.dtype], self.actions.element_size(), rows.data_ptr(), *strides,
            self.actions.data_ptr()))

    def results(self, *shape):
        return torch.empty(shape, dtype=torch.float32, device=self.device)

    def log_prob(self):
        log_prob, entropy = self.results(*self.shape), self.results(*self.shape)
        check(_library().mdn_op_choices_log_prob(ctypes.byref(self.c), log_prob.data_ptr(), entropy.data_ptr(),
                                                 _stream(self.device)))
        return log_prob, entropy


class _LossCall(_ChoiceCall):
    """The same with the loss's other arguments."""

    NAMES = ("old_log_prob", "advantages", "ref_log_prob", "mask")

    def __init__(self, logits, actions, old_log_prob, advantages, ref_log_prob, mask, low, high, kl_coef, entropy_coef):
        rows = (old_log_prob, advantages, ref_log_prob, mask)
        super().__init__(logits, actions, rows, self.NAMES)
        for name, t in zip(self.NAMES, rows):
            if t is None:
                continue
            _shape(name, t, self.shape)
            if name == "mask":
                if t.dtype not in (torch.uint8, torch.bool):
                    raise TypeError("mask is %s: uint8 or bool are taken" % t.dtype)
            elif t.dtype != torch.float32:
                raise TypeError("%s is %s: float32 is taken" % (name, t.dtype))
        self.rows = [None if t is None else t.contiguous() for t in rows]
        self.l = _ChoiceLoss.from_buffer_copy(_CHOICE_LOSS.pack(*(_address(t) or 0 for t in self.rows), low, high, kl_coef,
                                                                entropy_coef, 0, 0))

    def forward(self):
        L = _library()
        keep, work = ctypes.c_uint64(), ctypes.c_uint64()
        check(L.mdn_op_choices_loss_sizes(ctypes.byref(self.c), ctypes.byref(keep), ctypes.byref(work)))
        kept, buffer = _buffer(keep.value, self.device), _buffer(work.value, self.device)
        loss, metrics = self.results(), self.results(5)
        self.l.loss, self.l.metrics = loss.data_ptr(), metrics.data_ptr()
        check(L.mdn_op_choices_loss_forward(ctypes.byref(self.c), ctypes.byref(self.l), _address(kept), keep.value,
                                            _address(buffer), work.value, _stream(self.device)))
        return loss, metrics, kept

    def drop(self):
        self.logits = self.actions = self.rows = None

    def backward(self, kept, d_loss, logits):
        made = _like(logits)
        check(_library().mdn_op_choices_loss_backward(
            ctypes.byref(self.c), ctypes.byref(self.l), _address(kept), kept.numel(), d_loss.data_ptr(), made.data_ptr(),
            _stream(self.device)))
        return made


class _LossFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, actions, old_log_prob, advantages, ref_log_prob, mask, *numbers):
        call = _LossCall(logits, actions, old_log_prob, advantages, ref_log_prob, mask, *numbers)
        loss, metrics, kept = _on(call.device, call.forward)
        saved = (logits, actions, old_log_prob, advantages, ref_log_prob, mask)
        ctx.numbers, ctx.kept = numbers, _Kept(call, saved)
        ctx.save_for_backward(*saved, kept)
        ctx.mark_non_differentiable(metrics)
        ctx.set_materialize_grads(False)
        return loss, metrics

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_loss, _):
        if d_loss is None:
            return (None,) * 10
        *rows, kept = ctx.saved_tensors
        call = ctx.kept.again(rows) or _LossCall(*rows, *ctx.numbers)
        return (_on(call.device, call.backward, kept, d_loss.resolve_neg().contiguous(), rows[0]), *[None] * 9)


def _data(name, x):
    """Refuses a tensor that wants a gradient where there is none."""
    if isinstance(x, torch.Tensor) and x.requires_grad and torch.is_grad_enabled():
        raise TypeError("%s is data: it has no gradient here" % name)


def clipped_loss(logits, actions, old_log_prob, advantages, ref_log_prob=None, mask=None, clip=0.2, kl_coef=0.0,
                 entropy_coef=0.0):
    """The clipped loss of a policy over discrete choices: (loss, metrics).

    logits: [..., heads, choices], float32 or bfloat16: the independent choices
    of a step, four commands of so many levels or one of many manoeuvres, 1 to
    65,536 heads of below 2^24 choices.
    actions: [..., heads] int64 or int32.  old_log_prob, advantages,
    ref_log_prob: [...] float32, mask: [...] bool or uint8.  With l the sum of
    the heads' log-probabilities, H that of their entropies,
    r = exp(l - old_log_prob) and K = exp(ref_log_prob - l) -
    (ref_log_prob - l) - 1 (0 without ref_log_prob, and left out of the loss
    where kl_coef is 0), the loss is the mean of

        -min(r A, clip(r, 1 - low, 1 + high) A) + kl_coef K - entropy_coef H

    over the steps whose mask is set; ``clip`` is low and high alike, or a pair.
    metrics: the means of -min(..), K, H, r, and of r outside the borders.  No
    step that counts: all is 0.  Steps that do not count are not looked at, a
    logit of -inf rules a choice out, an action that is none of the choices
    gives NaN.  The gradient reaches the logits alone.
    """
    rows = (old_log_prob, advantages, ref_log_prob, mask)
    _tensors(logits=logits, actions=actions, old_log_prob=old_log_prob, advantages=advantages)
    _no_tangents(logits, *rows)
    for name, t in zip(_LossCall.NAMES, rows):
        _data(name, t)
    low, high = clip if isinstance(clip, (tuple, list)) else (clip, clip)
    for name, x in (("clip", low), ("clip", high), ("kl_coef", kl_coef), ("entropy_coef", entropy_coef)):
        _number(name, x)
    numbers = (float(low), float(high), float(kl_coef), float(entropy_coef))
    if not (numbers[0] >= 0.0 and numbers[1] >= 0.0):
        raise ValueError("clip is at least 0, not %r" % (clip,))
    if numbers[2] != 0.0 and ref_log_prob is None:
        raise ValueError("kl_coef needs ref_log_prob")
    if torch.is_grad_enabled() and isinstance(logits, torch.Tensor) and logits.requires_grad:
        return _LossFunction.apply(logits, actions, *rows, *numbers)
    call = _LossCall(logits, actions, *rows, *numbers)
    return _on(call.device, call.forward)[:2]


def log_prob(logits, actions):
    """(log-probability of the actions, entropy), summed over a step's heads, [...] float32: what acting stores.

    logits and actions as in ``clipped_loss``.  No gradients: logits that want
    one are refused.
    """
    _tensors(logits=logits, actions=actions)
    _no_tangents(logits)
    _data("logits", logits)
    call = _ChoiceCall(logits, actions)
    return _on(call.device, call.log_prob)
