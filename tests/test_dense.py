"""The linear layer and the gated feed-forward block (mdnav.policy) against their formulas in float64.

Tolerances, set before the first run, of the result's norm and past its own rounding.  u = 2^-24.  A sum of K products
is one fp32 chain; its roundings are relative to partial sums that grow like a random walk, which leaves
u sqrt(sum i / K) / sqrt(3) = 0.41 u sqrt(K), taken as u sqrt(K), and 16 u for what the epilogue does.  Activations
of bfloat16 rows use an exponential that is off by |z| u and, for gelu, an approximation of erf that is off by 1.5e-7:
both below 8 u in z's range here.  Gradients have dz, whose z and factors are off as the forward sums are, twice as
much where two are multiplied, and a sum over the other axis.  bfloat16 rows round dz once, at most 2^-8 of each value:
d_x and d_w may be off by that much of their norm."""
import ctypes
import math

import numpy as np
import pytest
import torch  # before the library: one HIP runtime in the process

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
LEAVES = ("x", "w", "w_up", "b", "b_up", "residual")


def erfc(x):
    return torch.erfc(x)


C = 2 * math.sqrt(2 / math.pi)
ACTS = {
    "none": (lambda z: z, lambda z: torch.ones_like(z)),
    "relu": (lambda z: torch.where(z > 0, z, 0 * z), lambda z: (z > 0).double()),
    "tanh": (torch.tanh, lambda z: 4 / (torch.exp(z) + torch.exp(-z)) ** 2),
    "sigmoid": (lambda z: 1 / (1 + torch.exp(-z)), lambda z: 1 / (1 + torch.exp(-z)) / (1 + torch.exp(z))),
    "silu": (lambda z: z / (1 + torch.exp(-z)), lambda z: (1 + z / (1 + torch.exp(z))) / (1 + torch.exp(-z))),
    "gelu": (lambda z: z * 0.5 * erfc(-z / math.sqrt(2)),
             lambda z: 0.5 * erfc(-z / math.sqrt(2)) + z * torch.exp(-z * z / 2) / math.sqrt(2 * math.pi)),
    "gelu_tanh": (lambda z: z / (1 + torch.exp(-C * (z + 0.044715 * z ** 3))),
                  lambda z: (1 + z * C * (1 + 0.134145 * z * z) / (1 + torch.exp(C * (z + 0.044715 * z ** 3))))
                  / (1 + torch.exp(-C * (z + 0.044715 * z ** 3)))),
}


def formula(v, act, d_y=None):
    """y, and with d_y every gradient, one step of the chain rule at a time; [rows][width] in float64."""
    f, slope = ACTS[act]

    def affine(w, b):
        z = torch.mm(v["x"], v[w].t().contiguous())
        return z if v.get(b) is None else z + v[b]

    z = affine("w", "b")
    up = affine("w_up", "b_up") if v.get("w_up") is not None else None
    y = f(z) if up is None else f(z) * up
    if v.get("residual") is not None:
        y = y + v["residual"]
    if d_y is None:
        return y, None
    dz = {"w": d_y * slope(z) if up is None else d_y * up * slope(z)}
    if up is not None:
        dz["w_up"] = d_y * f(z)
    g = dict(x=sum(torch.mm(d, v[n]) for n, d in dz.items()))
    for n, d in dz.items():
        g[n] = torch.mm(d.t().contiguous(), v["x"])
        if v.get("b" + n[1:]) is not None:
            g["b" + n[1:]] = d.sum(0)
    if v.get("residual") is not None:
        g["residual"] = d_y
    return y, g


def inputs(rows, width, out, dtype, gated, bias=True, residual=False, seed=0, device="cuda"):
    gen = torch.Generator().manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=gen, dtype=torch.float32)

    v = dict(x=randn(rows, width), w=randn(out, width) * width ** -0.5, w_up=randn(out, width) * width ** -0.5 if gated else None,
             b=0.3 * randn(out) if bias else None, b_up=0.3 * randn(out) if bias and gated else None,
             residual=randn(rows, out) if residual else None, d_y=randn(rows, out))
    return {n: None if t is None else t.to(dtype).to(device) for n, t in v.items()}


def call(v, act):
    from mdnav import policy
    if v.get("w_up") is not None:
        return policy.gated_feed_forward(v["x"], v["w"], v["w_up"], v.get("b"), v.get("b_up"), activation=act)
    return policy.linear(v["x"], v["w"], v.get("b"), activation=act, residual=v.get("residual"))


def near(name, got, want, room):
    low = got.dtype == BF16
    got = got.detach().double()
    assert got.shape == want.shape and torch.isfinite(got).all(), name
    if not want.numel():
        return
    rms = want.square().mean().sqrt()
    err = ((got - want).abs() - (2.0 ** -8 * want.abs() if low else 0.0)).clamp_(min=0)
    over = err.square().mean().sqrt()
    print("  %s: norm of the error past its rounding %.2e of %.2e" % (name, over / rms if rms else over, room), flush=True)
    assert over <= room * rms, (name, float(over / rms), room)
    assert (err <= 40 * room * torch.maximum(rms, want.abs())).all(), name


def rooms(rows, width, out, gated, dtype):
    z = U * (math.sqrt(width) + 16 + 8 * (dtype == BF16))
    dz = (3 if gated else 2) * z
    rounding = 2.0 ** -8 if dtype == BF16 else 0.0
    w = dz + U * math.sqrt(rows) + rounding
    b = dz + U * math.sqrt(rows)
    return dict(y=(2 if gated else 1) * z, x=dz + U * math.sqrt(out * (1 + gated)) + rounding, w=w, w_up=w, b=b, b_up=b,
                residual=0.0)


def check(v, act, dtype):
    leaves = {n: v[n].detach().requires_grad_() for n in LEAVES if v.get(n) is not None}
    y = call(dict(v, **leaves), act)
    assert y.dtype == dtype
    got = torch.autograd.grad(y, list(leaves.values()), v["d_y"])
    d = {n: None if t is None else t.double() for n, t in v.items()}
    want, grads = formula(d, act, d["d_y"])
    room = rooms(*v["x"].shape, v["w"].shape[0], v.get("w_up") is not None, dtype)
    if act == "none" and v.get("w_up") is None:  # (d_y is an operand as it is)
        room.update(x=room["x"] - 2.0 ** -8 * (dtype == BF16), w=room["w"] - 2.0 ** -8 * (dtype == BF16))
    near("y", y, want, room["y"])
    for (n, leaf), g in zip(leaves.items(), got):
        assert g.dtype == leaf.dtype and g.shape == leaf.shape
        near("d_" + n, g, grads[n], room[n])


@pytest.mark.parametrize("act", list(ACTS))
@pytest.mark.parametrize("gated", [False, True])
def test_the_gradients_here_match_differences(act, gated):
    v = {n: None if t is None else t.double() for n, t in inputs(4, 3, 5, F32, gated, residual=not gated, seed=3, device="cpu").items()}
    _, grads = formula(v, act, v["d_y"])
    for n, g in grads.items():
        for at in np.ndindex(tuple(v[n].shape)):
            values = []
            for step in (1e-6, -1e-6):
                t = v[n].clone()
                t[at] += step
                values.append((formula(dict(v, **{n: t}), act)[0] * v["d_y"]).sum())
            # values near 10 over 2e-6 in float64: 1e-9 of rounding, third derivatives up to 100 give 2e-11
            assert abs((values[0] - values[1]) / 2e-6 - g[at]) < 1e-7, (n, at)


# (on few rows; on small, middle and large tiles, with pieces of rows in dW and without; rows, widths and words that end inside)
SHAPES = [(1, 1, 1), (1, 64, 64), (7, 181, 33), (16, 128, 20), (17, 40, 48), (64, 184, 256), (130, 181, 70), (300, 184, 256),
          (257, 72, 129), (1000, 520, 130), (3001, 256, 333), (2000, 1032, 1024), (70001, 64, 256), (4097, 1024, 2056),
          (600, 3, 2), (129, 5120, 40)]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_matches_the_formula(shape, dtype):
    """Results and every gradient; activation, bias and residual go round with the shape."""
    kinds = list(ACTS)
    for i, gated in enumerate((False, True, False)):
        act = "none" if i == 2 else kinds[(sum(shape) + 3 * i) % len(kinds)]
        bias, residual = (sum(shape) + i) % 3 != 0, not gated and (sum(shape) + i) % 2 == 0
        print("case: dense", shape, dtype, gated, act, bias, residual, flush=True)
        check(inputs(*shape, dtype, gated, bias, residual, seed=sum(shape) + i), act, dtype)


@gpu
@pytest.mark.parametrize("rows", [5, 300])
@pytest.mark.parametrize("act", list(ACTS))
def test_activations_over_their_range(act, rows):
    """Values and slopes one by one, from -30 to 30: fp32 to 2^-20 of themselves down to 1e-30, bfloat16 to their
    rounding and, in gelu's tail, 2^-6 down to 1e-11.  The gelus' tails are exponentials of an argument e that is
    computed (z^2 / 2 by way of a rounded z / sqrt 2, sqrt(8 / pi) (z + 0.044715 z^3)): up to three roundings and a
    constant's, 4 u e of the value, with e = -log |value / z| near enough."""
    z = torch.linspace(-30, 30, rows * 16).reshape(rows, 16)
    for dtype in (F32, BF16):
        print("case: activation", act, rows, dtype, flush=True)
        x = z.to(dtype).cuda().requires_grad_()
        eye = torch.eye(16, dtype=dtype).cuda()
        y = call(dict(x=x, w=eye), act)
        slope, = torch.autograd.grad(y, x, torch.ones_like(y))
        f, g = ACTS[act]
        at = x.detach().double()
        for name, got, want in (("value", y, f(at)), ("slope", slope, g(at))):
            want = torch.where(torch.isnan(want), torch.zeros_like(want), want)
            room = 2.0 ** -20 if dtype == F32 else 2.0 ** -6 if act == "gelu" else 2.0 ** -7
            # where a slope passes 0 it is the difference of parts near 1
            low = 1e-30 if dtype == F32 and name == "value" else 1e-11
            if act.startswith("gelu"):
                room = room + 4 * U * torch.log((want / at).abs().clamp(1e-40, 1.0)).abs()
            allowed = room * want.abs() + (4 * U if name == "slope" or act == "tanh" else 0.0)
            big = want.abs() > low
            assert ((got.detach().double() - want).abs() <= allowed)[big].all(), name
            assert (got.detach().double().abs() <= 2 * low + 4 * U * (name == "slope"))[~big].all(), name


@gpu
@pytest.mark.parametrize("act,gated", [("silu", True), ("tanh", False), ("none", False)])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [24, 150])
def test_strides(rows, dtype, act, gated):
    """Operands in other layouts give the bits of contiguous ones, in results and gradients."""
    print("case: strides", rows, dtype, act, flush=True)
    v = inputs(rows, 40, 24, dtype, gated, residual=not gated, seed=9)
    leaves = [n for n in LEAVES if v[n] is not None]

    def run(t):
        t = {n: x.detach().requires_grad_() if n in leaves else x for n, x in t.items()}
        y = call(t, act)
        return [y] + list(torch.autograd.grad(y, [t[n] for n in leaves], t["d_y"]))

    def spread(t, gap, start):
        if t is None or t.dim() < 2:
            return t
        wide = torch.full((t.shape[0], t.shape[1] + gap + start), float("nan"), dtype=t.dtype, device="cuda")
        wide[:, start:start + t.shape[1]] = t
        return wide[:, start:start + t.shape[1]]

    want = run(v)
    for gap, start in ((8, 0), (7, 1), (3, 8)):
        for a, b in zip(run({n: spread(t, gap, start) for n, t in v.items()}), want):
            assert torch.equal(a, b)
    for a, b in zip(run({n: t if t is None or t.dim() < 2 else t.t().contiguous().t() for n, t in v.items()}), want):
        assert torch.equal(a, b)
    # two leading axes, exchanged in memory
    two = {n: v[n] if n in ("w", "w_up", "b", "b_up") or v[n] is None
           else v[n].unflatten(0, (3, -1)).transpose(0, 1).contiguous().transpose(0, 1) for n in v}
    for a, b in zip(run(two), want):
        assert torch.equal(a.reshape(b.shape), b)


@gpu
@pytest.mark.parametrize("act", ["none", "silu"])
def test_broadcast_inputs_and_gradients(act):
    """One row for all (a stride of 0), and a loss whose gradient is one number."""
    x = torch.randn(1, 40, generator=torch.Generator().manual_seed(2)).cuda().requires_grad_()
    w = torch.randn(24, 40, generator=torch.Generator().manual_seed(3)).cuda().requires_grad_()
    y = call(dict(x=x.expand(300, 40), w=w), act)
    got = torch.autograd.grad(y.sum(), [x, w])
    v = dict(x=x.detach().double().expand(300, 40), w=w.detach().double())
    want, g = formula(v, act, torch.ones_like(y, dtype=torch.float64))
    near("y", y, want, 30 * U)
    near("d_x", got[0], g["x"].sum(0, keepdim=True), 100 * U)
    near("d_w", got[1], g["w"], 100 * U)


@gpu
def test_a_residual_that_is_x():
    v = inputs(200, 64, 64, F32, False, residual=False, seed=4)
    x = v["x"].requires_grad_()
    y = call(dict(x=x, w=v["w"], residual=x), "gelu")
    got, = torch.autograd.grad(y, x, v["d_y"])
    d = {n: t.detach().double() for n, t in v.items() if t is not None}
    want, g = formula(dict(x=d["x"], w=d["w"], residual=d["x"]), "gelu", d["d_y"])
    near("y", y, want, 30 * U)
    near("d_x", got, g["x"] + g["residual"], 60 * U)


@gpu
@pytest.mark.parametrize("act,gated", [("silu", True), ("tanh", False), ("none", False)])
def test_gradients_that_are_asked_for(act, gated):
    """Each alone has the bits that it has with all."""
    v = inputs(333, 72, 40, BF16, gated, residual=not gated, seed=5)
    names = [n for n in LEAVES if v[n] is not None]

    def run(which):
        t = {n: x.detach().requires_grad_() if n in which else x for n, x in v.items()}
        return torch.autograd.grad(call(t, act), [t[n] for n in which], v["d_y"])

    for n, want in zip(names, run(names)):
        assert torch.equal(run([n])[0], want), n


@gpu
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("rows,width,out", [(20, 40, 24), (300, 40, 24), (5000, 520, 1024)])
def test_bad_rows_stay_alone(rows, width, out, bad):
    """A row that is not finite leaves the others' results and gradients as they are."""
    for dtype in (F32, BF16):
        print("case: bad row", rows, dtype, bad, flush=True)
        v = inputs(rows, width, out, dtype, True, seed=6)
        at = rows // 2
        worse = dict(v, x=v["x"].clone())
        worse["x"][at, width // 3] = bad
        got = []
        for t in (v, worse):
            x = t["x"].detach().requires_grad_()
            y = call(dict(t, x=x), "silu")
            got.append((y, torch.autograd.grad(y, x, t["d_y"])[0]))
        keep = torch.arange(rows) != at
        for a, b in zip(*got):
            assert torch.equal(a[keep], b[keep])
            assert not torch.isfinite(b[at]).all()


@gpu
def test_no_rows():
    for gated in (False, True):
        v = inputs(0, 40, 24, BF16, gated, seed=7)
        leaves = [v[n].requires_grad_() for n in LEAVES if v[n] is not None]
        y = call(v, "silu")
        assert y.shape == (0, 24)
        for leaf, g in zip(leaves, torch.autograd.grad(y, leaves, v["d_y"])):
            assert g.shape == leaf.shape and not g.any()


@gpu
def test_no_rows_through_the_c_entries():
    """The weights' and biases' gradients are zeros, between which nothing is written."""
    from mdnav import native, policy
    L = native.lib()
    v = inputs(0, 40, 30, BF16, True, seed=12)
    c = policy._Dense.from_buffer_copy(policy._DENSE.pack(
        0, 40, 30, 1, policy.ACTIVATIONS["silu"], 1, 0, 40, v["w"].data_ptr(), 40, v["w_up"].data_ptr(), 40, 0, 0, 0, 30, 0, 0))
    d_w, d_up = (torch.full((31, 44), 7.0, dtype=BF16, device="cuda") for _ in range(2))
    d_b, d_b_up = (torch.full((31,), 7.0, dtype=BF16, device="cuda") for _ in range(2))
    d = policy._DenseGrad.from_buffer_copy(policy._DENSE_GRAD.pack(0, 30, 0, 40, d_w.data_ptr(), 44, d_up.data_ptr(), 44,
                                                                   d_b.data_ptr(), d_b_up.data_ptr()))
    size = ctypes.c_uint64(9)
    stream = torch.cuda.current_stream().cuda_stream
    native.check(L.mdn_op_dense_forward(ctypes.byref(c), None, 0, stream))
    native.check(L.mdn_op_dense_backward_bytes(ctypes.byref(c), ctypes.byref(d), ctypes.byref(size)))
    assert size.value == 0
    native.check(L.mdn_op_dense_backward(ctypes.byref(c), ctypes.byref(d), None, 0, stream))
    for t in (d_w, d_up):
        assert not t[:30, :40].any() and (t[30:] == 7).all() and (t[:, 40:] == 7).all()
    for t in (d_b, d_b_up):
        assert not t[:30].any() and t[30] == 7


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_the_same_bits_every_time(dtype):
    v = inputs(20011, 200, 136, dtype, True, seed=8)
    runs = []
    for _ in range(3):
        leaves = [v[n].detach().requires_grad_() for n in LEAVES if v[n] is not None]
        y = call(dict(zip([n for n in LEAVES if v[n] is not None], leaves)), "gelu_tanh")
        runs.append([y] + list(torch.autograd.grad(y, leaves, v["d_y"])))
    for r in runs[1:]:
        for a, b in zip(r, runs[0]):
            assert torch.equal(a, b)


@gpu
def test_rows_past_four_gigabytes():
    """Rows 128 KB apart: offsets need more than 32 bits."""
    rows = 40000
    wide = torch.zeros(rows, 65536, dtype=BF16, device="cuda")
    v = inputs(rows, 16, 24, BF16, False, seed=11)
    wide[:, 32:48] = v["x"]
    x = wide[:, 32:48].requires_grad_()
    w = v["w"].requires_grad_()
    y = call(dict(v, x=x, w=w), "tanh")
    got = torch.autograd.grad(y, [x, w], v["d_y"])
    leaves = [v["x"].requires_grad_(), w]
    want = call(dict(v, w=w), "tanh")
    assert torch.equal(y, want)
    for a, b in zip(got, torch.autograd.grad(want, leaves, v["d_y"])):
        assert torch.equal(a, b)


@gpu
@pytest.mark.parametrize("gated", [False, True])
def test_what_was_saved_may_move(gated):
    """Saved tensors that a hook brings back elsewhere, or as a view of more, give the same gradients; so does a weight
    whose memory is another by then."""
    v = inputs(300, 40, 48, BF16, gated, seed=15)
    names = [n for n in LEAVES if v[n] is not None]
    leaves = {n: v[n].clone().requires_grad_() for n in names}
    want = torch.autograd.grad(call(dict(v, **leaves), "silu"), list(leaves.values()), v["d_y"])
    for back in (lambda t: t.clone(), lambda t: torch.cat((t, t), -1)[..., :t.shape[-1]]):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: back(t.cuda())):
            y = call(dict(v, **leaves), "silu")
        for a, b in zip(torch.autograd.grad(y, list(leaves.values()), v["d_y"]), want):
            assert torch.equal(a, b)
    y = call(dict(v, **leaves), "silu")
    old = leaves["w"].data
    leaves["w"].data = old.clone()
    old.fill_(math.nan)
    for a, b in zip(torch.autograd.grad(y, list(leaves.values()), v["d_y"]), want):
        assert torch.equal(a, b)


@gpu
def test_more_rows_than_a_launch_has_small_tiles():
    """2^30 rows, all the same one: 2^24 tiles of 64 rows would be 2^32 threads."""
    from mdnav import policy
    v = inputs(64, 8, 64, BF16, False, seed=14)
    y = policy.linear(v["x"][:1].expand(1 << 30, 8), v["w"], v["b"], "silu")
    want = policy.linear(v["x"], v["w"], v["b"], "silu")[:1]
    for at in (0, (1 << 29) - 500, (1 << 30) - 1000):
        # sums of 8 in another order, at most one step of the result
        torch.testing.assert_close(y[at:at + 1000].float(), want.expand(1000, 64).float(), rtol=2.0 ** -7, atol=1e-6)


@gpu
@pytest.mark.parametrize("rows", [20, 500])
def test_only_the_results_are_written(rows):
    """Results with rows apart, through the C entries: what lies between stays."""
    from mdnav import native, policy
    L = native.lib()
    v = inputs(rows, 40, 30, BF16, True, seed=12)
    y = torch.full((rows + 2, 44), 7.0, dtype=BF16, device="cuda")
    d_x = torch.full((rows + 2, 52), 7.0, dtype=BF16, device="cuda")
    d_w = torch.full((32, 52), 7.0, dtype=BF16, device="cuda")

    def matrix(t, width, row=0):
        return t[row].data_ptr(), width

    c = policy._Dense.from_buffer_copy(policy._DENSE.pack(
        rows, 40, 30, 1, policy.ACTIVATIONS["silu"], 1, *matrix(v["x"], 40), *matrix(v["w"], 40), *matrix(v["w_up"], 40), 0, 0,
        *matrix(y, 44, 1), v["b"].data_ptr(), v["b_up"].data_ptr()))
    d = policy._DenseGrad.from_buffer_copy(policy._DENSE_GRAD.pack(*matrix(v["d_y"], 30), *matrix(d_x, 52, 1), *matrix(d_w, 52, 1),
                                                                   0, 0, 0, 0))
    size = ctypes.c_uint64()
    stream = torch.cuda.current_stream().cuda_stream
    native.check(L.mdn_op_dense_forward_bytes(ctypes.byref(c), ctypes.byref(size)))
    work = torch.empty(size.value + 1, dtype=torch.uint8, device="cuda")
    native.check(L.mdn_op_dense_forward(ctypes.byref(c), work.data_ptr(), size.value, stream))
    native.check(L.mdn_op_dense_backward_bytes(ctypes.byref(c), ctypes.byref(d), ctypes.byref(size)))
    work = torch.empty(size.value + 1, dtype=torch.uint8, device="cuda")
    native.check(L.mdn_op_dense_backward(ctypes.byref(c), ctypes.byref(d), work.data_ptr(), size.value, stream))
    leaves = [v["x"].requires_grad_(), v["w"].requires_grad_()]
    want = call(v, "silu")
    g = torch.autograd.grad(want, leaves, v["d_y"])
    for wide, inner, width in ((y, want, 30), (d_x, g[0], 40), (d_w, g[1], 40)):
        n = inner.shape[0]
        assert torch.equal(wide[1:n + 1, :width], inner)
        assert (wide[0] == 7).all() and (wide[n + 1:] == 7).all() and (wide[:, width:] == 7).all()


@gpu
@pytest.mark.parametrize("rows", [9, 700])
def test_captured_graphs_and_streams(rows):
    """Two graphs of forward and backward calls, replayed in turn between eager calls, and a call on another stream."""
    from mdnav import policy
    v = inputs(rows, 72, 40, BF16, True, seed=13)
    names = [n for n in LEAVES if v[n] is not None]
    gen = torch.Generator(device="cuda").manual_seed(3)

    def fill():
        for n in names:
            v[n].copy_(torch.randn(v[n].shape, generator=gen, device="cuda") * 0.2)

    def calls():
        t = {n: v[n].detach().requires_grad_() for n in names}
        y = call(t, "silu")
        return [y.detach()] + list(torch.autograd.grad(y, list(t.values()), v["d_y"]))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, calls()))
    for i in range(4):
        fill()
        want = [t.clone() for t in calls()]
        graph, captured = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = calls()
        torch.cuda.current_stream().wait_stream(side)
        for a, b in zip(beside, want):
            assert torch.equal(a, b)


# ---------------------------------------------------------------- refusals
@pytest.fixture
def on_the_cpu(monkeypatch):
    from mdnav import policy
    monkeypatch.setattr(policy, "_device", lambda names, tensors: torch.device("cpu"))

    def reached(*args):
        raise AssertionError("the library was called")

    monkeypatch.setattr(policy, "_library", reached)
    monkeypatch.setattr(policy, "_on", lambda device, f, *args: f(*args))
    return policy


def test_refusals(on_the_cpu):
    policy, z = on_the_cpu, torch.zeros
    x, w, b = z(5, 8), z(6, 8), z(6)
    for args, more, error, text in [
            ((x, z(6, 7)), {}, ValueError, "x has shape"), ((x, z(6)), {}, ValueError, "weight is"),
            ((x, w, z(5)), {}, ValueError, "bias has shape"), ((x, w, b), dict(residual=z(5, 8)), ValueError, "residual has shape"),
            ((x, w.bfloat16()), {}, TypeError, "one type"), ((x.double(), w.double()), {}, TypeError, "float32 or bfloat16"),
            ((x, w, b.bfloat16()), {}, TypeError, "one type"), ((x, w), dict(activation="swish"), ValueError, "activation is one of"),
            ((z(()), w), {}, ValueError, "x is"), ((z(5, 0), z(6, 0)), {}, ValueError, "widths"),
            ((z(1, 8), z(65537, 8)), {}, ValueError, "widths"), ((x, w), dict(residual=z(6)), ValueError, "residual has shape")]:
        with pytest.raises(error, match=text):
            policy.linear(*args, **more)
    for args, error, text in [((x, w, z(6, 7)), ValueError, "w_up has shape"), ((x, w, z(5, 8)), ValueError, "w_up has shape"),
                              ((x, w, None), TypeError, "w_up is no tensor"), ((x, w, w, b, z(7)), ValueError, "b_up has shape")]:
        with pytest.raises(error, match=text):
            policy.gated_feed_forward(*args)
    with pytest.raises(AssertionError, match="was called"):
        policy.linear(x, w, b, activation="gelu", residual=z(5, 6))


def test_tensors_elsewhere_are_refused():
    from mdnav import policy
    import torch.autograd.forward_ad as forward_ad
    x, w = torch.zeros(3, 4), torch.zeros(5, 4)
    for f in (lambda: policy.linear(x, w), lambda: policy.gated_feed_forward(x, w, w)):
        with pytest.raises(ValueError, match="not on a GPU"):
            f()
    with pytest.raises(TypeError, match="is no tensor"):
        policy.linear(x, None)
    with forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            policy.linear(forward_ad.make_dual(x, x), w)
        with pytest.raises(NotImplementedError, match="forward-mode"):
            policy.gated_feed_forward(x, w, forward_ad.make_dual(w, w))


def test_the_c_entries_refuse_before_anything_runs():
    from mdnav import native, policy
    L = native.lib()
    good = dict(rows=3, in_=8, out=8, dtype=0, activation=0, gated=0)

    def dense(**more):
        c = policy._Dense()
        for n, x in dict(good, **more).items():
            if n in ("x", "w", "w_up", "residual", "y"):
                getattr(c, n).data = x
            else:
                setattr(c, n, x)
        for n in ("x", "w", "y"):
            if n not in more:
                getattr(c, n).data = 4096
            getattr(c, n).row = 8
        return c

    size = ctypes.c_uint64()
    for more, text in [(dict(dtype=2), b"dtype"), (dict(activation=7), b"activation"), (dict(gated=2), b"gated"), (dict(in_=0), b"1..65536"),
                       (dict(out=65537), b"1..65536"), (dict(rows=1 << 31), b"too many rows"), (dict(w=None), b"null weights"),
                       (dict(x=None), b"null rows"), (dict(gated=1), b"null weights"), (dict(w_up=4096), b"gated block"),
                       (dict(gated=1, w_up=4096, residual=4096), b"no residual"), (dict(b_up=4096), b"gated block")]:
        c = dense(**more)
        assert L.mdn_op_dense_forward_bytes(ctypes.byref(c), ctypes.byref(size)) == -1 and text in L.mdn_last_error(), more
        assert L.mdn_op_dense_forward(ctypes.byref(c), None, 0, None) == -1 and text in L.mdn_last_error(), more
    assert L.mdn_op_dense_forward_bytes(None, ctypes.byref(size)) == -1
    c = dense(y=None)
    assert L.mdn_op_dense_forward(ctypes.byref(c), None, 0, None) == -1 and b"null rows" in L.mdn_last_error()
    # rows that are no whole words are copied: the workspace is asked for, and checked
    c = dense(rows=1000, in_=7)
    assert L.mdn_op_dense_forward_bytes(ctypes.byref(c), ctypes.byref(size)) == 0 and size.value >= 1000 * 8 * 4
    assert L.mdn_op_dense_forward(ctypes.byref(c), None, 0, None) == -1 and b"workspace" in L.mdn_last_error()
    assert L.mdn_op_dense_forward(ctypes.byref(c), 4100, size.value, None) == -1 and b"aligned" in L.mdn_last_error()
    d = policy._DenseGrad()
    c = dense(rows=1000)
    assert L.mdn_op_dense_backward(ctypes.byref(c), None, None, 0, None) == -1
    assert L.mdn_op_dense_backward(ctypes.byref(c), ctypes.byref(d), None, 0, None) == -1 and b"null rows" in L.mdn_last_error()
    d.d_y.data, d.d_y.row, d.d_w_up.data = 4096, 8, 4096
    assert L.mdn_op_dense_backward(ctypes.byref(c), ctypes.byref(d), None, 0, None) == -1 and b"gated block" in L.mdn_last_error()
    d.d_w_up.data, d.d_b = None, 4096
    assert L.mdn_op_dense_backward_bytes(ctypes.byref(c), ctypes.byref(d), ctypes.byref(size)) == 0 and size.value > 0
    assert L.mdn_op_dense_backward(ctypes.byref(c), ctypes.byref(d), None, 0, None) == -1 and b"workspace" in L.mdn_last_error()
    assert L.mdn_op_dense_backward(ctypes.byref(c), ctypes.byref(d), 4100, size.value, None) == -1 and b"aligned" in L.mdn_last_error()
