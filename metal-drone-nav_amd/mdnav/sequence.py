"""Operators of recurrent policies over torch tensors on the GPU: the gated
delta rule, whole rollouts with gradients (``delta_rule``) and one tick of a
fleet in place (``delta_rule_step``), and the norms around a block
(``block_norm``).

Unlike ``ops``, which copies numpy arrays to the device and back, these take
device tensors as they are, run on torch's current stream and return device
tensors.  Rows are time-major, [ticks][envs][heads][width], as the rollout
buffers are; any strides go as long as the width is contiguous, so
``x.transpose(0, 1)`` of batch-first rows needs no copy.  An argument that is a
lazily negated view (``is_neg()``, of a conjugate's imaginary part) is to be
resolved before; a gradient that arrives as one is resolved here.

torch is imported here and nowhere else in the package, and it has to be
imported before the library is first used: both need the same HIP runtime in
the process, and the one loaded first is taken.
"""
import ctypes
import struct

import torch
import torch.autograd.forward_ad as forward_ad
import torch.autograd.function

from .native import MdnError, P, check, lib

F32, BF16 = 0, 1
_DTYPES = {torch.float32: F32, torch.bfloat16: BF16}


class _Rows(ctypes.Structure):
    _fields_ = [("data", P), ("tick", ctypes.c_int64), ("env", ctypes.c_int64), ("head", ctypes.c_int64)]


class _DeltaRule(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint32) for n in ("ticks", "envs", "qk_heads", "heads", "k_dim", "v_dim", "dtype",
                                               "gate_dtype")]
    _fields_ += [("scale", ctypes.c_float)]
    _fields_ += [(n, _Rows) for n in ("q", "k", "v", "g", "beta", "o")]
    _fields_ += [("reset", P), ("reset_tick", ctypes.c_int64), ("reset_env", ctypes.c_int64), ("state", P),
                 ("state_out", P)]


class _DeltaRuleGrad(ctypes.Structure):
    _fields_ = [("d_o", _Rows), ("d_state_out", P)]
    _fields_ += [(n, _Rows) for n in ("d_q", "d_k", "d_v", "d_g", "d_beta")]
    _fields_ += [("d_state", P)]


class _Sizes(ctypes.Structure):
    _fields_ = [(n, ctypes.c_uint64) for n in ("keep", "forward_workspace", "backward_workspace")]


class _NormRows(ctypes.Structure):
    _fields_ = [("data", P), ("outer", ctypes.c_int64), ("inner", ctypes.c_int64)]


class _BlockNorm(ctypes.Structure):
    _fields_ = [("rows", ctypes.c_uint64)]
    _fields_ += [(n, ctypes.c_uint32) for n in ("inner_count", "width", "x_dtype", "y_dtype", "gate_kind", "gate_dtype")]
    _fields_ += [("epsilon", ctypes.c_float)]
    _fields_ += [(n, _NormRows) for n in ("x", "y", "gate", "s", "h")]
    _fields_ += [(n, P) for n in ("w_post", "w_pre", "residual", "stats")]


class _BlockNormGrad(ctypes.Structure):
    _fields_ = [(n, _NormRows) for n in ("d_s", "d_h", "d_x", "d_y", "d_gate")]
    _fields_ += [(n, P) for n in ("d_w_post", "d_w_pre", "d_residual")]


# The structs as packed bytes, made of plain numbers in one call each: 2.2 us
# for a tick's, where nested ctypes objects took 4.1.
_RULE = struct.Struct("=8If4x29q")
_RULE_GRAD = struct.Struct("=26q")
_ROWS = struct.Struct("=4q")
_NORM = struct.Struct("=Q6If4x19q")
_NORM_OUT = struct.Struct("=6q")
_NORM_GRAD = struct.Struct("=18q")
assert _RULE.size == ctypes.sizeof(_DeltaRule) and _NORM.size == ctypes.sizeof(_BlockNorm)
assert _RULE_GRAD.size == ctypes.sizeof(_DeltaRuleGrad) and _NORM_GRAD.size == ctypes.sizeof(_BlockNormGrad)

_one_runtime = None


def _library():
    """The library, once it is known to share torch's HIP runtime: streams and
    memory of another runtime in the process would not be the same."""
    global _one_runtime
    L = lib()
    if _one_runtime is None:
        with open("/proc/self/maps") as f:
            paths = {line.split()[-1] for line in f if "libamdhip64.so" in line}
        _one_runtime = len(paths) <= 1
    if not _one_runtime:
        raise MdnError("two HIP runtimes are loaded: import torch before the first use of mdnav's library")
    return L


def _device(names, tensors):
    """The GPU that all tensors are on."""
    try:
        index = tensors[0].get_device()  # (half the time of as many comparisons of devices)
        if index >= 0 and all([t is None or t.get_device() == index for t in tensors]):
            return tensors[0].device
    except AttributeError:
        pass
    device = None  # which one is not
    for name, t in zip(names, tensors):
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError("%s is no tensor" % name)
        if device is None:
            device = t.device
            if device.type != "cuda":
                raise ValueError("%s is not on a GPU" % name)
        elif t.device != device:
            raise ValueError("%s is on %s, other arguments on %s" % (name, t.device, device))
    return device


def _no_tangents(*tensors):
    """Forward-mode derivatives, which there are none of here: the kernels see a dual tensor's value alone, and a
    result without a tangent would read as a derivative of zero."""
    if forward_ad._current_level < 0:
        return
    for t in tensors:
        if isinstance(t, torch.Tensor) and forward_ad.unpack_dual(t).tangent is not None:
            raise NotImplementedError("forward-mode derivatives are not available, only gradients")


def _number(name, x):
    """Refuses a tensor that wants the gradient which a plain number has none of."""
    if isinstance(x, torch.Tensor) and x.requires_grad and torch.is_grad_enabled():
        raise TypeError("%s is a number: it has no gradient" % name)


def _on(device, call, *args):
    """call(*args) with `device` the current GPU."""
    if torch.cuda.current_device() == device.index:
        return call(*args)
    with torch.cuda.device(device):
        return call(*args)


def _stream(device):
    # torch.cuda.current_stream(device).cuda_stream without the object around it: 0.1 and not 1.9 us of a call
    return torch._C._cuda_getCurrentRawStream(device.index)


def _like(t):
    return torch.empty_like(t, memory_format=torch.contiguous_format)


def _address(t):
    return None if t is None else t.data_ptr()


def _buffer(size, device):
    return torch.empty(size, dtype=torch.uint8, device=device) if size else None


def _wide(t):
    """The tensor with a contiguous width."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _shape(name, t, shape):
    if t.shape != shape:
        raise ValueError("%s has shape %s, expected %s" % (name, tuple(t.shape), tuple(shape)))


def _rows(t, one_tick=False):
    """A [ticks][envs][heads][width] (or, gates, [ticks][envs][heads]) tensor; `one_tick`: without the ticks."""
    strides = t.stride()
    return (t.data_ptr(), 0, strides[0], strides[1]) if one_tick else (t.data_ptr(), *strides[:3])


class _Call:
    """Checked arguments of one delta rule call: the C struct and what it points to."""

    NAMES = ("q", "k", "v", "g", "beta", "state", "reset")

    def __init__(self, q, k, v, g, beta, state, reset, scale, one_tick=False):
        self.device = _device(self.NAMES, (q, k, v, g, beta, state, reset))
        lead = 1 if one_tick else 2
        if q.dim() != lead + 2 or v.dim() != lead + 2:
            raise ValueError("q, k and v are %s[envs][heads][width]" % ("" if one_tick else "[ticks]"))
        sq, sv = q.shape, v.shape
        hq, kd = sq[lead:]
        h, vd = sv[lead:]
        t, n = (1, sq[0]) if one_tick else sq[:2]
        _shape("k", k, sq)
        _shape("v", v, (*sq[:lead], h, vd))
        _shape("g", g, sv[:-1])
        _shape("beta", beta, sv[:-1])
        if hq < 1 or h < 1 or h % hq:
            raise ValueError("%d query heads do not divide %d value heads" % (hq, h))
        if not 1 <= kd <= 128 or not 1 <= vd <= 128:
            raise ValueError("head widths are 1..128, not %d and %d" % (kd, vd))
        dtype = q.dtype
        if dtype not in _DTYPES:
            raise TypeError("q is %s: float32 or bfloat16 are taken" % dtype)
        if k.dtype != dtype or v.dtype != dtype:
            raise TypeError("q is %s, k %s and v %s: one type is taken" % (dtype, k.dtype, v.dtype))
        if g.dtype != beta.dtype or g.dtype not in (torch.float32, dtype):
            raise TypeError("g and beta are float32 or both of q's type, not %s and %s" % (g.dtype, beta.dtype))
        if reset is not None:
            _shape("reset", reset, sq[:lead])
            if reset.dtype not in (torch.uint8, torch.bool):
                raise TypeError("reset is %s: uint8 or bool are taken" % reset.dtype)
        if state is not None:
            _shape("state", state, (n, h, kd, vd))
            if state.dtype != torch.float32:
                raise TypeError("state is %s: float32 is taken" % state.dtype)
        self.q, self.k, self.v, self.g, self.beta = _wide(q), _wide(k), _wide(v), g, beta
        self.state, self.reset = state, reset
        first = (0, 0, 0)
        if reset is not None:
            first = (reset.data_ptr(), 0, reset.stride(0)) if one_tick else (reset.data_ptr(), *reset.stride())
        self.c = _DeltaRule.from_buffer_copy(_RULE.pack(
            t, n, hq, h, kd, vd, _DTYPES[dtype], _DTYPES[g.dtype], kd ** -0.5 if scale is None else scale,
            *_rows(self.q, one_tick), *_rows(self.k, one_tick), *_rows(self.v, one_tick), *_rows(g, one_tick),
            *_rows(beta, one_tick), 0, 0, 0, 0, *first, 0 if state is None else state.data_ptr(), 0))

    def output(self):
        return _like(self.v)

    def states(self):
        c = self.c
        return torch.empty(c.envs, c.heads, c.k_dim, c.v_dim, dtype=torch.float32, device=self.device)

    def forward(self, o, state_out, keep):
        """One call over all ticks; `keep`: whether a backward pass follows.  What that reads, and its workspace."""
        L = _library()
        c = self.c
        _ROWS.pack_into(c, _DeltaRule.o.offset, *_rows(o))
        c.state_out = _address(state_out)
        sizes = _Sizes()
        check(L.mdn_op_delta_rule_sizes(ctypes.byref(c), ctypes.byref(sizes)))
        kept = _buffer(sizes.keep, self.device) if keep else None
        work = _buffer(sizes.forward_workspace, self.device)
        check(L.mdn_op_delta_rule_forward(ctypes.byref(c), _address(kept), sizes.keep if keep else 0, _address(work),
                                          sizes.forward_workspace, _stream(self.device)))
        return kept, sizes

    def step(self, o, state):
        """One tick, which needs no buffers."""
        c = self.c
        _ROWS.pack_into(c, _DeltaRule.o.offset, *_rows(o, True))
        c.state_out = state.data_ptr()
        check(_library().mdn_op_delta_rule_forward(ctypes.byref(c), None, 0, None, 0, _stream(self.device)))

    def backward(self, kept, sizes, d_o, d_state_out, want_state):
        """(d_q, d_k, d_v, d_g, d_beta, d_state or None)"""
        grads = [_like(x) for x in (self.q, self.k, self.v, self.g, self.beta)]
        d_state = self.states() if want_state else None
        work = _buffer(sizes.backward_workspace, self.device)
        dq, dk, dv, dg, db = [_rows(x) for x in grads]
        d = _DeltaRuleGrad.from_buffer_copy(_RULE_GRAD.pack(
            *_rows(d_o), 0 if d_state_out is None else d_state_out.data_ptr(), *dq, *dk, *dv, *dg, *db,
            0 if d_state is None else d_state.data_ptr()))
        check(_library().mdn_op_delta_rule_backward(ctypes.byref(self.c), ctypes.byref(d), _address(kept), sizes.keep,
                                                    _address(work), sizes.backward_workspace, _stream(self.device)))
        return (*grads, d_state)


class _DeltaRuleFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, reset, scale, final_state):
        call = _Call(q, k, v, g, beta, state, reset, scale)
        o, last = call.output(), call.states() if final_state else None
        kept, ctx.sizes = _on(call.device, call.forward, o, last, True)
        ctx.scale = scale
        ctx.save_for_backward(q, k, v, g, beta, state, reset, kept)
        ctx.set_materialize_grads(False)
        return o, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_last):
        if d_o is None and d_last is None:
            return (None,) * 9
        q, k, v, g, beta, state, reset, kept = ctx.saved_tensors
        d_o = torch.zeros_like(v) if d_o is None else _wide(d_o.resolve_neg())
        d_last = None if d_last is None else d_last.resolve_neg().contiguous()
        want_state = state is not None and ctx.needs_input_grad[5]
        if q.shape[0] == 0:  # nothing happens to the state
            d_state = None if not want_state else torch.zeros_like(state) if d_last is None else d_last
            return (*[torch.zeros_like(x) for x in (q, k, v, g, beta)], d_state, None, None, None)
        call = _Call(q, k, v, g, beta, state, reset, ctx.scale)
        return (*_on(call.device, call.backward, kept, ctx.sizes, d_o, d_last, want_state), None, None, None)


def delta_rule(q, k, v, g, beta, state=None, reset=None, scale=None, final_state=False):
    """The gated delta rule over whole rollouts: (o, final state or None).

    Per environment and head, with a state S of K x V in 32 bits:
    S <- 0 where ``reset`` is set, S <- exp(g) S, u = beta (v - S^T k),
    S <- S + k u^T, o = scale S^T q.

    q, k: [ticks][envs][qk heads][K], v: [ticks][envs][heads][V], float32 or
    bfloat16; the query heads divide the value heads and are shared by
    consecutive ones.  g (log decay, -inf allowed) and beta:
    [ticks][envs][heads], float32 or of q's type.  reset: [ticks][envs] uint8 or
    bool.  state: [envs][heads][K][V] float32 before the first tick (zeros if
    None).  scale: K ** -0.5 if None.  o has v's shape and q's type.  Gradients
    reach every tensor argument but reset; a flagged tick has none for g.

    The state is held in 32 bits.  Products of float32 rows are float32; with
    bfloat16 rows the state and what else is computed enter products with 16
    to 17 bits, with all 24 where ``final_state`` is asked for (o then differs
    by roundings to bfloat16 that fall on the other side), and gradients with
    16 to 17, those in float32 (state, float32 g and beta) too.  A g below
    -104 clears the state as ``reset`` does; the g of a flagged tick is not
    looked at.
    """
    _no_tangents(q, k, v, g, beta, state, scale)
    _number("scale", scale)
    if isinstance(state, torch.Tensor):
        state = state.contiguous()
    if torch.is_grad_enabled() and any(isinstance(x, torch.Tensor) and x.requires_grad for x in (q, k, v, g, beta, state)):
        return _DeltaRuleFunction.apply(q, k, v, g, beta, state, reset, scale, final_state)
    call = _Call(q, k, v, g, beta, state, reset, scale)
    o, last = call.output(), call.states() if final_state else None
    _on(call.device, call.forward, o, last, False)
    return o, last


def delta_rule_step(q, k, v, g, beta, state, reset=None, scale=None):
    """One tick of a fleet: o, with ``state`` advanced in place.

    q, k: [envs][qk heads][K], v: [envs][heads][V], g, beta: [envs][heads],
    reset: [envs], state: contiguous [envs][heads][K][V] float32; otherwise as
    ``delta_rule``.  No gradients: autograd sees ``state`` change, as by any
    operation in place, so a backward pass that still reads the old one raises.
    """
    _no_tangents(q, k, v, g, beta, state, scale)
    _number("scale", scale)
    if not isinstance(state, torch.Tensor) or not state.is_contiguous():
        raise ValueError("state is a contiguous tensor: it is advanced in place")
    if state.requires_grad and torch.is_grad_enabled():
        raise ValueError("state requires gradients, which a tick in place has none for")
    call = _Call(q, k, v, g, beta, state, reset, scale, one_tick=True)
    o = call.output()
    _on(call.device, call.step, o, state)
    torch.autograd.graph.increment_version(state)
    return o


# ---------------------------------------------------------------- norms around a block
GATE_NONE, GATE_CHANNEL, GATE_ROW, GATE_ELEMENT = 0, 1, 2, 3


class _NormCall:
    """Checked arguments of one norm block call."""

    NAMES = ("x", "y", "w_post", "w_pre", "gate", "residual_scale")

    def __init__(self, x, y, w_post, w_pre, gate, residual_scale, eps):
        self.device = _device(self.NAMES, (x, y, w_post, w_pre, gate, residual_scale))
        shape = x.shape
        if len(shape) < 1:
            raise ValueError("x is [..., width]")
        _shape("y", y, shape)
        width = shape[-1]
        if not 1 <= width <= 8192:
            raise ValueError("the width is 1..8192, not %d" % width)
        if x.dtype not in _DTYPES or y.dtype not in _DTYPES or (x.dtype == torch.bfloat16 and y.dtype == torch.float32):
            raise TypeError("x and y are float32, both bfloat16, or float32 and bfloat16, not %s and %s" % (x.dtype, y.dtype))
        for name, w in (("w_post", w_post), ("w_pre", w_pre), ("residual_scale", residual_scale)):
            if w is None and name == "residual_scale":
                continue
            _shape(name, w, (width,))
            if w.dtype != torch.float32:
                raise TypeError("%s is %s: float32 is taken" % (name, w.dtype))
        self.kind = GATE_NONE
        if gate is not None:
            if gate.dtype != torch.float32 and gate.dtype != y.dtype:
                raise TypeError("gate is %s: float32 or y's type are taken" % gate.dtype)
            if gate.shape == (width,) and (len(shape) > 1 or width > 1):
                self.kind = GATE_CHANNEL
                gate = gate.contiguous()
            elif gate.shape == (*shape[:-1], 1):
                self.kind = GATE_ROW
            elif gate.shape == shape:
                self.kind = GATE_ELEMENT
                if gate.dtype != y.dtype:
                    raise TypeError("a gate per element is of y's type, %s, not %s" % (y.dtype, gate.dtype))
            else:
                raise ValueError("gate has shape %s, expected %s, %s or %s" % (
                    tuple(gate.shape), (width,), (*shape[:-1], 1), tuple(shape)))
        self.x, self.y, self.gate = x, y, gate
        self.w_post, self.w_pre = w_post.contiguous(), w_pre.contiguous()
        self.residual = None if residual_scale is None else residual_scale.contiguous()
        self.shape, self.width, self.rows = shape, width, x.numel() // width
        self.inner = shape[-2] if len(shape) > 1 and self.rows else 1
        self.kept = []  # copies that the struct points to
        rows = (0, 0, 0) if gate is None else (gate.data_ptr(), 0, 0) if self.kind == GATE_CHANNEL else self.layout(gate)
        self.c = _BlockNorm.from_buffer_copy(_NORM.pack(
            self.rows, self.inner, width, _DTYPES[x.dtype], _DTYPES[y.dtype], self.kind, 0 if gate is None else _DTYPES[gate.dtype],
            eps, *self.layout(x), *self.layout(y), *rows, 0, 0, 0, 0, 0, 0, self.w_post.data_ptr(), self.w_pre.data_ptr(),
            0 if self.residual is None else self.residual.data_ptr(), 0))

    def layout(self, t):
        """The rows of `t`, [..., width or 1], as two strides; another layout is copied."""
        if not t.is_contiguous():
            axes = [] if t.shape[-1] == 1 or t.stride(-1) == 1 else None
            if axes is not None:
                # join neighbouring axes that are one
                for size, stride in zip(t.shape[:-1], t.stride()[:-1]):
                    if size == 1:
                        continue
                    if axes and axes[-1][1] == size * stride:
                        axes[-1] = (axes[-1][0] * size, stride)
                    else:
                        axes.append((size, stride))
                if len(axes) <= 1:
                    stride = axes[0][1] if axes else 0
                    return t.data_ptr(), stride * self.inner, stride
                if len(axes) == 2 and axes[1][0] == self.inner:
                    return t.data_ptr(), axes[0][1], axes[1][1]
            t = t.contiguous()
            self.kept.append(t)
        return t.data_ptr(), t.shape[-1] * self.inner, t.shape[-1]

    def made(self, t):
        """The layout of a contiguous [..., width] tensor."""
        return t.data_ptr(), self.width * self.inner, self.width

    def forward(self, keep):
        L = _library()
        s, h = _like(self.x), _like(self.y)
        stats = torch.empty(self.rows, 2, dtype=torch.float32, device=self.device) if keep else None
        c = self.c
        _NORM_OUT.pack_into(c, _BlockNorm.s.offset, *self.made(s), *self.made(h))
        c.stats = _address(stats)
        check(L.mdn_op_block_norm_forward(ctypes.byref(c), _stream(self.device)))
        return s, h, stats

    def backward(self, stats, d_s, d_h):
        L = _library()
        c, none = self.c, (0, 0, 0)
        c.stats = _address(stats)
        d_x, d_y = _like(self.x), _like(self.y)
        d_gate, gate = None, none
        if self.kind != GATE_NONE:
            d_gate = _like(self.gate)
            gate = self.layout(d_gate) if self.kind != GATE_CHANNEL else (d_gate.data_ptr(), 0, 0)
        d_post, d_pre, d_scale = torch.empty(3, self.width, dtype=torch.float32, device=self.device).unbind()
        if self.residual is None:
            d_scale = None
        d = _BlockNormGrad.from_buffer_copy(_NORM_GRAD.pack(
            *(none if d_s is None else self.layout(d_s)), *(none if d_h is None else self.layout(d_h)), *self.made(d_x),
            *self.made(d_y), *gate, d_post.data_ptr(), d_pre.data_ptr(), 0 if d_scale is None else d_scale.data_ptr()))
        size = ctypes.c_uint64()
        check(L.mdn_op_block_norm_workspace_bytes(ctypes.byref(c), ctypes.byref(size)))
        work = _buffer(size.value, self.device)
        check(L.mdn_op_block_norm_backward(ctypes.byref(c), ctypes.byref(d), _address(work), size.value, _stream(self.device)))
        return d_x, d_y, d_post, d_pre, d_gate, d_scale


class _BlockNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, w_post, w_pre, gate, residual_scale, eps):
        call = _NormCall(x, y, w_post, w_pre, gate, residual_scale, eps)
        s, h, stats = _on(call.device, call.forward, True)
        ctx.eps = eps
        ctx.save_for_backward(x, y, w_post, w_pre, gate, residual_scale, stats)
        ctx.set_materialize_grads(False)
        return s, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_s, d_h):
        if d_s is None and d_h is None:
            return (None,) * 7
        d_s, d_h = (None if d is None else d.resolve_neg() for d in (d_s, d_h))
        x, y, w_post, w_pre, gate, residual_scale, stats = ctx.saved_tensors
        call = _NormCall(x, y, w_post, w_pre, gate, residual_scale, ctx.eps)
        return (*_on(call.device, call.backward, stats, d_s, d_h), None)


def block_norm(x, y, w_post, w_pre, gate=None, residual_scale=None, eps=1e-6):
    """The norms around a block, with its gate and residual scale: (s, h).

    n = y / rms(y), s = residual_scale x + gate n w_post, h = s / rms(s) w_pre:
    x is the residual stream [..., width], y the block's output, s the stream
    after it and h the next block's input.  x and y are float32, both bfloat16,
    or float32 and bfloat16; s has x's type, h has y's.  w_post, w_pre and
    residual_scale (ones if None) are [width] float32.  gate (ones if None):
    [width], one value per row [..., 1], or one per element, float32 or, per
    element always, of y's type.  Gradients reach every tensor argument.
    """
    args = (x, y, w_post, w_pre, gate, residual_scale)
    _no_tangents(*args, eps)
    _number("eps", eps)
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in args):
        return _BlockNormFunction.apply(*args, eps)
    call = _NormCall(*args, eps)
    return _on(call.device, call.forward, False)[:2]
