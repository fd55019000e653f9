"""Operators of recurrent policies over torch tensors on the GPU: the gated
delta rule, whole rollouts with gradients (``delta_rule``) and one tick of a
fleet in place (``delta_rule_step``), and the norms around a block
(``block_norm``).

Unlike ``ops``, which copies numpy arrays to the device and back, these take
device tensors as they are, run on torch's current stream and return device
tensors.  Rows are time-major, [ticks][envs][heads][width], as the rollout
buffers are; any strides go as long as the width is contiguous, so
``x.transpose(0, 1)`` of batch-first rows needs no copy.

torch is imported here and nowhere else in the package, and it has to be
imported before the library is first used: both need the same HIP runtime in
the process, and the one loaded first is taken.
"""
import ctypes

import torch
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


def _device(named):
    """The GPU that all tensors are on."""
    device = None
    for name, t in named:
        if t is None:
            continue
        if not isinstance(t, torch.Tensor):
            raise TypeError("%s is no tensor" % name)
        if not t.is_cuda:
            raise ValueError("%s is not on a GPU" % name)
        if device is None:
            device = t.device
        elif t.device != device:
            raise ValueError("%s is on %s, other arguments on %s" % (name, t.device, device))
    return device


def _rows(t):
    """A [ticks][envs][heads][width] (or, gates, [ticks][envs][heads]) tensor."""
    return _Rows(t.data_ptr(), t.stride(0), t.stride(1), t.stride(2))


def _wide(t):
    """The tensor with a contiguous width."""
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _shape(name, t, shape):
    if tuple(t.shape) != tuple(shape):
        raise ValueError("%s has shape %s, expected %s" % (name, tuple(t.shape), tuple(shape)))


class _Call:
    """Checked arguments of one delta rule call: the C struct and what it points to."""

    def __init__(self, q, k, v, g, beta, state, reset, scale):
        self.device = _device([("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta), ("state", state),
                               ("reset", reset)])
        if q.dim() != 4 or v.dim() != 4:
            raise ValueError("q, k and v are [ticks][envs][heads][width]")
        t, n, hq, kd = q.shape
        h, vd = v.shape[2:]
        _shape("k", k, q.shape)
        _shape("v", v, (t, n, h, vd))
        _shape("g", g, (t, n, h))
        _shape("beta", beta, (t, n, h))
        if hq < 1 or h < 1 or h % hq:
            raise ValueError("%d query heads do not divide %d value heads" % (hq, h))
        if not 1 <= kd <= 128 or not 1 <= vd <= 128:
            raise ValueError("head widths are 1..128, not %d and %d" % (kd, vd))
        if q.dtype not in _DTYPES:
            raise TypeError("q is %s: float32 or bfloat16 are taken" % q.dtype)
        for name, x in (("k", k), ("v", v)):
            if x.dtype != q.dtype:
                raise TypeError("%s is %s, q is %s" % (name, x.dtype, q.dtype))
        if g.dtype != beta.dtype or g.dtype not in (torch.float32, q.dtype):
            raise TypeError("g and beta are float32 or both of q's type, not %s and %s" % (g.dtype, beta.dtype))
        if reset is not None:
            _shape("reset", reset, (t, n))
            if reset.dtype not in (torch.uint8, torch.bool):
                raise TypeError("reset is %s: uint8 or bool are taken" % reset.dtype)
        if state is not None:
            _shape("state", state, (n, h, kd, vd))
            if state.dtype != torch.float32:
                raise TypeError("state is %s: float32 is taken" % state.dtype)
        self.q, self.k, self.v = _wide(q), _wide(k), _wide(v)
        self.g, self.beta, self.state, self.reset = g, beta, state, reset
        self.scale = kd ** -0.5 if scale is None else float(scale)
        c = _DeltaRule(t, n, hq, h, kd, vd, _DTYPES[q.dtype], _DTYPES[g.dtype], self.scale, _rows(self.q),
                       _rows(self.k), _rows(self.v), _rows(g), _rows(beta))
        if reset is not None:
            c.reset, c.reset_tick, c.reset_env = reset.data_ptr(), reset.stride(0), reset.stride(1)
        if state is not None:
            c.state = state.data_ptr()
        self.c = c

    def stream(self):
        return torch.cuda.current_stream(self.device).cuda_stream

    def bytes_of(self, function, *more):
        size = ctypes.c_uint64()
        check(function(ctypes.byref(self.c), *more, ctypes.byref(size)))
        return size.value

    def buffer(self, size):
        return torch.empty(size, dtype=torch.uint8, device=self.device) if size else None


def _address(t):
    return None if t is None else t.data_ptr()


def _forward(call, o, state_out, keep):
    """One forward call; `keep`: whether a backward pass follows."""
    L = _library()
    call.c.o = _rows(o)
    call.c.state_out = _address(state_out)
    with torch.cuda.device(call.device):
        kept = call.buffer(call.bytes_of(L.mdn_op_delta_rule_keep_bytes)) if keep else None
        size = call.bytes_of(L.mdn_op_delta_rule_workspace_bytes, 0)
        work = call.buffer(size)
        check(L.mdn_op_delta_rule_forward(ctypes.byref(call.c), _address(kept), 0 if kept is None else kept.numel(),
                                          _address(work), size, call.stream()))
    return kept


def _backward(call, kept, d_o, d_state_out, want_state):
    """(d_q, d_k, d_v, d_g, d_beta, d_state or None)"""
    L = _library()
    c = call.c
    with torch.cuda.device(call.device):
        grads = [torch.empty(x.shape, dtype=x.dtype, device=x.device) for x in (call.q, call.k, call.v, call.g, call.beta)]
        d_state = torch.empty(c.envs, c.heads, c.k_dim, c.v_dim, device=call.device) if want_state else None
        size = call.bytes_of(L.mdn_op_delta_rule_workspace_bytes, 1)
        work = call.buffer(size)
        d = _DeltaRuleGrad(_rows(d_o), _address(d_state_out), *[_rows(x) for x in grads], _address(d_state))
        check(L.mdn_op_delta_rule_backward(ctypes.byref(c), ctypes.byref(d), _address(kept),
                                           0 if kept is None else kept.numel(), _address(work), size, call.stream()))
    return (*grads, d_state)


class _DeltaRuleFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, g, beta, state, reset, scale, final_state):
        call = _Call(q, k, v, g, beta, state, reset, scale)
        o = torch.empty(v.shape, dtype=v.dtype, device=v.device)
        last = _final_state(call) if final_state else None
        kept = _forward(call, o, last, True)
        ctx.scale, ctx.has_state = scale, state is not None
        ctx.save_for_backward(q, k, v, g, beta, state, reset, kept)
        ctx.set_materialize_grads(False)
        return o, last

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_o, d_last):
        q, k, v, g, beta, state, reset, kept = ctx.saved_tensors
        if d_o is None and d_last is None:
            return (None,) * 9
        call = _Call(q, k, v, g, beta, state, reset, ctx.scale)
        d_o = torch.zeros_like(v) if d_o is None else _wide(d_o)
        want_state = ctx.has_state and ctx.needs_input_grad[5]
        if q.shape[0] == 0:  # nothing happens to the state
            d_state = None if not want_state else torch.zeros_like(state) if d_last is None else d_last
            return (*[torch.zeros_like(x) for x in (q, k, v, g, beta)], d_state, None, None, None)
        grads = _backward(call, kept, d_o, None if d_last is None else d_last.contiguous(), want_state)
        return (*grads, None, None, None)


def _final_state(call):
    c = call.c
    return torch.empty(c.envs, c.heads, c.k_dim, c.v_dim, device=call.device)


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
    """
    state = None if state is None else state.contiguous()
    if torch.is_grad_enabled() and any(x is not None and x.requires_grad for x in (q, k, v, g, beta, state)):
        return _DeltaRuleFunction.apply(q, k, v, g, beta, state, reset, scale, final_state)
    call = _Call(q, k, v, g, beta, state, reset, scale)
    o = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    last = _final_state(call) if final_state else None
    _forward(call, o, last, False)
    return o, last


def delta_rule_step(q, k, v, g, beta, state, reset=None, scale=None):
    """One tick of a fleet: o, with ``state`` advanced in place.

    q, k: [envs][qk heads][K], v: [envs][heads][V], g, beta: [envs][heads],
    reset: [envs], state: contiguous [envs][heads][K][V] float32; otherwise as
    ``delta_rule``.  No gradients.
    """
    if not isinstance(state, torch.Tensor) or not state.is_contiguous():
        raise ValueError("state is a contiguous tensor: it is advanced in place")
    call = _Call(q[None], k[None], v[None], g[None], beta[None], state, None if reset is None else reset[None], scale)
    o = torch.empty(v.shape, dtype=v.dtype, device=v.device)
    _forward(call, o[None], state, False)
    return o


# ---------------------------------------------------------------- norms around a block
GATE_NONE, GATE_CHANNEL, GATE_ROW, GATE_ELEMENT = 0, 1, 2, 3


def _norm_rows(t, width):
    """A tensor whose last axis is a row, as two strides: (tensor, rows, count of the inner axis)."""
    t = t if t.shape[-1] == 1 or t.stride(-1) == 1 else t.contiguous()
    lead, strides = t.shape[:-1], t.stride()[:-1]
    # join neighbouring axes that are one; at most two may remain
    axes = []
    for size, stride in zip(lead, strides):
        if size == 1:
            continue
        if axes and axes[-1][1] == size * stride:
            axes[-1] = (axes[-1][0] * size, stride)
        else:
            axes.append((size, stride))
    return t, axes


class _NormCall:
    """Checked arguments of one norm block call."""

    def __init__(self, x, y, w_post, w_pre, gate, residual_scale, eps):
        self.device = _device([("x", x), ("y", y), ("w_post", w_post), ("w_pre", w_pre), ("gate", gate),
                               ("residual_scale", residual_scale)])
        if x.dim() < 1:
            raise ValueError("x is [..., width]")
        _shape("y", y, x.shape)
        width = x.shape[-1]
        if not 1 <= width <= 8192:
            raise ValueError("the width is 1..8192, not %d" % width)
        if x.dtype not in _DTYPES or y.dtype not in _DTYPES or (x.dtype, y.dtype) == (torch.bfloat16, torch.float32):
            raise TypeError("x and y are float32, both bfloat16, or float32 and bfloat16, not %s and %s" % (x.dtype, y.dtype))
        for name, w in (("w_post", w_post), ("w_pre", w_pre), ("residual_scale", residual_scale)):
            if w is None and name == "residual_scale":
                continue
            _shape(name, w, (width,))
            if w.dtype != torch.float32:
                raise TypeError("%s is %s: float32 is taken" % (name, w.dtype))
        self.kind = GATE_NONE
        if gate is not None:
            if gate.dtype not in (torch.float32, y.dtype):
                raise TypeError("gate is %s: float32 or y's type are taken" % gate.dtype)
            if tuple(gate.shape) == (width,) and (x.dim() > 1 or width > 1):
                self.kind = GATE_CHANNEL
            elif tuple(gate.shape) == tuple(x.shape[:-1]) + (1,):
                self.kind = GATE_ROW
            elif tuple(gate.shape) == tuple(x.shape):
                self.kind = GATE_ELEMENT
                if gate.dtype != y.dtype:
                    raise TypeError("a gate per element is of y's type, %s, not %s" % (y.dtype, gate.dtype))
            else:
                raise ValueError("gate has shape %s, expected %s, %s or %s" % (
                    tuple(gate.shape), (width,), tuple(x.shape[:-1]) + (1,), tuple(x.shape)))
        self.x, self.y, self.gate = x, y, gate
        self.w_post, self.w_pre = w_post.contiguous(), w_pre.contiguous()
        self.residual = None if residual_scale is None else residual_scale.contiguous()
        self.shape, self.width, self.rows, self.eps = x.shape, width, x.numel() // width, float(eps)
        self.inner = x.shape[-2] if x.dim() > 1 and self.rows else 1

    def layout(self, t):
        """The rows of `t`, [..., width or 1]; a layout of more than two strides is copied."""
        t, axes = _norm_rows(t, self.width)
        if not axes:
            return t, _NormRows(t.data_ptr(), 0, 0)
        if len(axes) == 1:
            return t, _NormRows(t.data_ptr(), axes[0][1] * self.inner, axes[0][1])
        if len(axes) == 2 and axes[1][0] == self.inner:
            return t, _NormRows(t.data_ptr(), axes[0][1], axes[1][1])
        t = t.contiguous()
        return t, _NormRows(t.data_ptr(), t.shape[-1] * self.inner, t.shape[-1])

    def struct(self, s, h, stats):
        """The C struct, and the tensors it points to."""
        kept = [s, h, stats]
        c = _BlockNorm(self.rows, self.inner, self.width, _DTYPES[self.x.dtype], _DTYPES[self.y.dtype], self.kind,
                       0 if self.gate is None else _DTYPES[self.gate.dtype], self.eps)
        for name in ("x", "y"):
            t, rows = self.layout(getattr(self, name))
            kept.append(t)
            setattr(c, name, rows)
        if self.kind == GATE_CHANNEL:
            t = self.gate.contiguous()
            kept.append(t)
            c.gate = _NormRows(t.data_ptr(), 0, 0)
        elif self.kind != GATE_NONE:
            t, c.gate = self.layout(self.gate)
            kept.append(t)
        if s is not None:
            c.s, c.h = self.layout(s)[1], self.layout(h)[1]
        c.w_post, c.w_pre = self.w_post.data_ptr(), self.w_pre.data_ptr()
        c.residual, c.stats = _address(self.residual), _address(stats)
        return c, kept

    def forward(self, keep):
        L = _library()
        s = torch.empty(self.shape, dtype=self.x.dtype, device=self.device)
        h = torch.empty(self.shape, dtype=self.y.dtype, device=self.device)
        stats = torch.empty(self.rows, 2, device=self.device) if keep else None
        with torch.cuda.device(self.device):
            c, kept = self.struct(s, h, stats)
            check(L.mdn_op_block_norm_forward(ctypes.byref(c), torch.cuda.current_stream().cuda_stream))
        return s, h, stats

    def backward(self, stats, d_s, d_h):
        L = _library()
        with torch.cuda.device(self.device):
            c, kept = self.struct(None, None, stats)
            d = _BlockNormGrad()
            for name, t in (("d_s", d_s), ("d_h", d_h)):
                if t is not None:
                    t, rows = self.layout(t)
                    kept.append(t)
                    setattr(d, name, rows)
            d_x = torch.empty(self.shape, dtype=self.x.dtype, device=self.device)
            d_y = torch.empty(self.shape, dtype=self.y.dtype, device=self.device)
            d.d_x, d.d_y = self.layout(d_x)[1], self.layout(d_y)[1]
            d_gate = None
            if self.kind != GATE_NONE:
                d_gate = torch.empty(self.gate.shape, dtype=self.gate.dtype, device=self.device)
                d.d_gate = _NormRows(d_gate.data_ptr(), 0, 0) if self.kind == GATE_CHANNEL else self.layout(d_gate)[1]
            sums = torch.empty(2 if self.residual is None else 3, self.width, device=self.device)
            d.d_w_post, d.d_w_pre = sums[0].data_ptr(), sums[1].data_ptr()
            if self.residual is not None:
                d.d_residual = sums[2].data_ptr()
            size = ctypes.c_uint64()
            check(L.mdn_op_block_norm_workspace_bytes(ctypes.byref(c), ctypes.byref(size)))
            work = torch.empty(size.value, dtype=torch.uint8, device=self.device) if size.value else None
            check(L.mdn_op_block_norm_backward(ctypes.byref(c), ctypes.byref(d), _address(work), size.value,
                                               torch.cuda.current_stream().cuda_stream))
        return d_x, d_y, sums[0], sums[1], d_gate, None if self.residual is None else sums[2]


class _BlockNormFunction(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, y, w_post, w_pre, gate, residual_scale, eps):
        s, h, stats = _NormCall(x, y, w_post, w_pre, gate, residual_scale, eps).forward(True)
        ctx.eps = eps
        ctx.save_for_backward(x, y, w_post, w_pre, gate, residual_scale, stats)
        ctx.set_materialize_grads(False)
        return s, h

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, d_s, d_h):
        x, y, w_post, w_pre, gate, residual_scale, stats = ctx.saved_tensors
        if d_s is None and d_h is None:
            return (None,) * 7
        return (*_NormCall(x, y, w_post, w_pre, gate, residual_scale, ctx.eps).backward(stats, d_s, d_h), None)


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
    if torch.is_grad_enabled() and any(isinstance(t, torch.Tensor) and t.requires_grad for t in args):
        return _BlockNormFunction.apply(*args, eps)
    return _NormCall(*args, eps).forward(False)[:2]
