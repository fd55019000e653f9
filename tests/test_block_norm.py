"""The norm block (mdnav.sequence.block_norm) against its formula in float64.

Tolerances, set before the first run.  Rows are fp32 arithmetic on at most
8,192 terms per sum, formed as 64 or more lanes' partial sums (at most 128
terms in a row, then a tree of ten): 140 roundings of 2^-24 at worst, 8.3e-6 of
the norm, of which random signs leave less than a tenth; taken as 1e-6.  A
bfloat16 result is rounded once more, at most 2^-8 of its value.  Column sums
add at most 64 rows in a lane, 16 lanes and 1,024 / 4 workgroups in a row, 340
roundings of 2^-24: 2.0e-5 of the sum of magnitudes at worst; against the
norm of the sums, where random signs make rounding and sum grow alike, taken
as 4e-6."""
import numpy as np
import pytest
import torch  # before the library: one HIP runtime in the process

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16


def formula(x, y, w_post, w_pre, gate=None, residual_scale=None, eps=1e-6):
    g = 1.0 if gate is None else gate
    r = 1.0 if residual_scale is None else residual_scale
    n = y / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
    s = r * x + g * (n * w_post)
    return s, s / np.sqrt((s * s).mean(-1, keepdims=True) + eps) * w_pre


def gradients(x, y, w_post, w_pre, gate, residual_scale, d_s, d_h, eps=1e-6):
    """By the chain rule from the formula, one step at a time."""
    g = np.ones(1) if gate is None else gate
    r = np.ones(x.shape[-1]) if residual_scale is None else residual_scale
    ry = 1.0 / np.sqrt((y * y).mean(-1, keepdims=True) + eps)
    n = y * ry
    b = n * w_post
    s = r * x + g * b
    rs = 1.0 / np.sqrt((s * s).mean(-1, keepdims=True) + eps)
    lead = tuple(range(x.ndim - 1))
    z = d_h * w_pre
    d_sum = d_s + rs * z - s * rs ** 3 * (z * s).mean(-1, keepdims=True)
    d_n = d_sum * g * w_post
    out = dict(x=d_sum * r, y=ry * d_n - y * ry ** 3 * (d_n * y).mean(-1, keepdims=True),
               w_post=(d_sum * g * n).sum(lead), w_pre=(d_h * s * rs).sum(lead))
    if gate is not None:
        whole = d_sum * b
        out["gate"] = (whole.sum(lead) if gate.ndim == 1 else whole if gate.shape == x.shape
                       else whole.sum(-1, keepdims=True))
    if residual_scale is not None:
        out["residual_scale"] = (d_sum * x).sum(lead)
    return out


@pytest.mark.parametrize("kind", ["none", "channel", "row", "element"])
def test_the_gradients_here_match_differences(kind):
    rng = np.random.default_rng(4)
    shape = (3, 2, 5)
    gate = dict(none=None, channel=(5,), row=(3, 2, 1), element=shape)[kind]
    x = dict(x=rng.normal(size=shape), y=rng.normal(size=shape), w_post=rng.normal(size=5), w_pre=rng.normal(size=5),
             gate=None if gate is None else rng.normal(size=gate),
             residual_scale=None if kind == "none" else rng.normal(size=5))
    d_s, d_h = rng.normal(size=shape), rng.normal(size=shape)
    grads = gradients(**x, d_s=d_s, d_h=d_h)

    def value(z):
        s, h = formula(**z)
        return (s * d_s).sum() + (h * d_h).sum()

    for name, array in x.items():
        if array is None:
            continue
        for at in np.ndindex(array.shape):
            z = {m: None if a is None else a.copy() for m, a in x.items()}
            z[name][at] += 1e-6
            up = value(z)
            z[name][at] -= 2e-6
            # values near 10 over 2e-6 in float64: 1e-9 of rounding, third derivatives up to 100 give 2e-11
            assert abs((up - value(z)) / 2e-6 - grads[name][at]) < 1e-7, (name, at)


def near(name, got, want, room):
    low = got.dtype == BF16
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape and np.isfinite(got).all(), name
    if not want.size:
        return
    rms = np.sqrt(np.mean(want ** 2))
    err = np.maximum(np.abs(got - want) - (2.0 ** -8 * np.abs(want) if low else 0.0), 0.0)
    over = np.sqrt(np.mean(err ** 2))
    print("  %s: norm of the error past its rounding %.2e" % (name, over / rms if rms else over), flush=True)
    assert over <= room * rms, (name, over / rms)
    assert np.all(err <= 40 * room * np.maximum(rms, np.abs(want))), name


def inputs(shape, kind, x_type, y_type, residual=True, seed=0, gate_type=None):
    gen = torch.Generator().manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=gen)

    width = shape[-1]
    gate = dict(none=None, channel=(width,), row=tuple(shape[:-1]) + (1,), element=tuple(shape))[kind]
    gate_type = gate_type or (y_type if kind in ("element", "row") else F32)
    x = dict(x=randn(*shape).to(x_type), y=(0.5 * randn(*shape) + 0.1).to(y_type), w_post=1 + 0.1 * randn(width),
             w_pre=1 + 0.1 * randn(width), gate=None if gate is None else torch.sigmoid(randn(*gate)).to(gate_type),
             residual_scale=1 + 0.1 * randn(width) if residual else None)
    d_s, d_h = randn(*shape).to(x_type), randn(*shape).to(y_type)
    return {n: None if t is None else t.cuda() for n, t in x.items()}, d_s.cuda(), d_h.cuda()


def host(x):
    return {n: None if t is None else t.detach().double().cpu().numpy() for n, t in x.items()}


TYPES = {"f32": (F32, F32), "bf16": (BF16, BF16), "mixed": (F32, BF16)}
SHAPES = [(1, 1), (2, 3, 1), (5, 64), (1, 181), (37, 181), (16, 7, 256), (3, 1000), (300, 24), (33, 129), (6, 513), (7, 2049),
          (4, 5120), (2, 8191), (3, 8192), (1100, 33)]


@gpu
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_matches_the_formula(shape, types):
    """Both results and every gradient; the kind of gate goes round with the shape."""
    from mdnav import sequence
    for kind in ("none", "channel", "row", "element"):
        if kind == "channel" and shape[-1] == 1 or kind in ("row", "element") and shape[-1] == 1 and kind == "row":
            continue  # one channel: a gate per channel, row and element have shapes of their own below
        print("case: block_norm", shape, types, kind, flush=True)
        x, d_s, d_h = inputs(shape, kind, *TYPES[types], residual=kind != "none", seed=sum(shape))
        leaves = {n: t.requires_grad_() for n, t in x.items() if t is not None}
        s, h = sequence.block_norm(**x)
        assert s.dtype == TYPES[types][0] and h.dtype == TYPES[types][1]
        got = torch.autograd.grad([s, h], list(leaves.values()), [d_s, d_h])
        v = host(x)
        want_s, want_h = formula(**v)
        near("s", s, want_s, 1e-6)
        near("h", h, want_h, 1e-6)
        want = gradients(**v, d_s=d_s.double().cpu().numpy(), d_h=d_h.double().cpu().numpy())
        for (n, leaf), grad in zip(leaves.items(), got):
            assert grad.dtype == leaf.dtype and grad.shape == leaf.shape
            near("d_" + n, grad, want[n], 4e-6 if n.startswith("w") or n == "residual_scale" or (n, kind) == ("gate", "channel") else 1e-6)


@gpu
def test_without_gradients_gives_the_same_results():
    from mdnav import sequence
    x, _, _ = inputs((20, 200), "element", BF16, BF16)
    s, h = sequence.block_norm(**x)
    x["x"].requires_grad_()
    s2, h2 = sequence.block_norm(**x)
    assert torch.equal(s, s2) and torch.equal(h, h2) and s2.requires_grad


@gpu
@pytest.mark.parametrize("width", [64, 40, 181])
def test_strides(width):
    """Rows of other tensors: transposed, cut, broadcast, unaligned and reversed axes of three."""
    from mdnav import sequence
    gen = torch.Generator().manual_seed(width)
    big = torch.randn(4, 3, 5, width + 11, generator=gen).cuda()
    flat = torch.randn(3 * 5 * width + 1, generator=gen).cuda()
    w = torch.ones(width).cuda()
    views = dict(cut=big[0, :, :, 3:3 + width], turned=big[1].transpose(0, 1)[:, :, :width], one=big[2, :1, :1, 1:1 + width],
                 broadcast=big[0, :, :1, :width].expand(3, 5, width), shifted=flat[1:].view(3, 5, width),
                 three=big.permute(2, 0, 1, 3)[:, :, :, :width], columns=big[0, :, :, ::2][..., :(width + 11) // 2])
    for name, x in views.items():
        print("case: strides", name, tuple(x.shape), x.stride(), flush=True)
        ww = w[:x.shape[-1]]
        y = torch.randn(x.shape, generator=gen).cuda()
        for a, b in ((x, y), (y, x)):
            s, h = sequence.block_norm(a, b, ww, ww)
            s2, h2 = sequence.block_norm(a.contiguous(), b.contiguous(), ww, ww)
            assert torch.equal(s, s2) and torch.equal(h, h2), name


@gpu
def test_broadcast_gate_and_shared_inputs():
    """A gate expanded over the ticks gets the sum of its gradients; a tensor used twice gets both."""
    from mdnav import sequence
    x, d_s, d_h = inputs((6, 5, 32), "none", F32, F32, residual=False)
    gate = torch.rand(1, 5, 1, generator=torch.Generator().manual_seed(1)).cuda().requires_grad_()
    x["x"].requires_grad_()
    s, h = sequence.block_norm(x["x"], x["x"], x["w_post"], x["w_pre"], gate=gate.expand(6, 5, 1))
    d_x, d_gate = torch.autograd.grad([s, h], [x["x"], gate], [d_s, d_h])
    v = host(x)
    want = gradients(v["x"], v["x"], v["w_post"], v["w_pre"], np.broadcast_to(gate.detach().double().cpu().numpy(), (6, 5, 1)),
                     None, d_s.double().cpu().numpy(), d_h.double().cpu().numpy())
    near("d_x", d_x, want["x"] + want["y"], 1e-6)
    near("d_gate", d_gate, want["gate"].sum(0, keepdims=True), 4e-6)


@gpu
def test_one_result_unused():
    from mdnav import sequence
    x, d_s, d_h = inputs((9, 70), "channel", F32, F32)
    zero = np.zeros((9, 70))
    for which in (0, 1):
        leaves = {n: t.detach().requires_grad_() for n, t in x.items()}
        out = sequence.block_norm(**leaves)
        got = torch.autograd.grad(out[which], list(leaves.values()), (d_s, d_h)[which], allow_unused=True)
        want = gradients(**host(x), d_s=d_s.double().cpu().numpy() if which == 0 else zero,
                         d_h=d_h.double().cpu().numpy() if which == 1 else zero)
        for n, grad in zip(leaves, got):
            near("d_" + n, grad, want[n], 4e-6) if want[n].any() else None
            assert grad is None or torch.isfinite(grad).all()


@gpu
def test_no_rows():
    from mdnav import sequence
    x, d_s, d_h = inputs((0, 4, 16), "channel", BF16, BF16)
    leaves = {n: t.requires_grad_() for n, t in x.items()}
    s, h = sequence.block_norm(**x)
    assert s.shape == h.shape == (0, 4, 16)
    got = dict(zip(leaves, torch.autograd.grad([s, h], list(leaves.values()), [d_s, d_h])))
    assert all(got[n].shape == x[n].shape for n in got)
    for n in ("w_post", "w_pre", "gate", "residual_scale"):
        assert not got[n].any()


@gpu
def test_rows_do_not_meet():
    """A row of NaN or infinities leaves the others as they were, column sums aside."""
    from mdnav import sequence
    x, d_s, d_h = inputs((40, 64), "element", F32, F32)
    s, h = sequence.block_norm(**x)
    x["y"][7] = float("nan")
    x["x"][21, 3] = float("inf")
    x["y"][30] = 0.0
    s2, h2 = sequence.block_norm(**x)
    rows = [r for r in range(40) if r not in (7, 21, 30)]
    assert torch.equal(s[rows], s2[rows]) and torch.equal(h[rows], h2[rows])
    assert torch.isnan(s2[7]).all() and torch.isinf(s2[21, 3])
    assert torch.equal(s2[30], x["residual_scale"] * x["x"][30])  # a row of zeros stays zeros


@gpu
def test_same_bits_every_time():
    from mdnav import sequence
    x, d_s, d_h = inputs((5000, 96), "row", BF16, BF16)
    leaves = [t.requires_grad_() for t in x.values()]
    runs = []
    for _ in range(2):
        out = sequence.block_norm(**x)
        runs.append(list(out) + list(torch.autograd.grad(out, leaves, [d_s, d_h])))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


def test_refusals():
    """Arguments the operator has no meaning for, before anything is launched."""
    from mdnav import sequence
    x, w = torch.zeros(3, 8), torch.ones(8)
    with pytest.raises(ValueError, match="GPU"):
        sequence.block_norm(x, x, w, w)
    with pytest.raises(TypeError, match="no tensor"):
        sequence.block_norm([1.0], x, w, w)


@gpu
def test_refusals_on_the_gpu():
    from mdnav import sequence
    x, w = torch.zeros(3, 8).cuda(), torch.ones(8).cuda()
    for bad, error, match in (
            (lambda: sequence.block_norm(x, x[:2], w, w), ValueError, "y has shape"),
            (lambda: sequence.block_norm(x, x, w[:7], w), ValueError, "w_post"),
            (lambda: sequence.block_norm(x, x, w, w.double()), TypeError, "w_pre"),
            (lambda: sequence.block_norm(x.half(), x.half(), w, w), TypeError, "float16"),
            (lambda: sequence.block_norm(x.bfloat16(), x, w, w), TypeError, "bfloat16"),
            (lambda: sequence.block_norm(x, x, w, w, gate=w[:5]), ValueError, "gate has shape"),
            (lambda: sequence.block_norm(x, x, w, w, gate=x.bfloat16()), TypeError, "gate"),
            (lambda: sequence.block_norm(x, x.bfloat16(), w, w, gate=x), TypeError, "gate per element"),
            (lambda: sequence.block_norm(x, x, w, w, residual_scale=x), ValueError, "residual_scale"),
            (lambda: sequence.block_norm(torch.zeros(1, 8193).cuda(), torch.zeros(1, 8193).cuda(), w, w), ValueError, "8192")):
        with pytest.raises(error, match=match):
            bad()


def test_the_c_entries_refuse():
    """What the C entries check themselves, before anything is launched."""
    import ctypes
    from mdnav import native, sequence
    lib = native.lib()
    some = 4096
    good = sequence._BlockNorm(3, 1, 64, 0, 0, 1, 0, 1e-6)
    for name in ("x", "y", "gate", "s", "h"):
        getattr(good, name).data = some
    good.w_post = good.w_pre = good.stats = some

    def refused(text, **fields):
        c = sequence._BlockNorm.from_buffer_copy(good)
        for name, value in fields.items():
            setattr(c, name, value)
        assert lib.mdn_op_block_norm_forward(ctypes.byref(c), None) == -1
        assert text in lib.mdn_last_error().decode(), lib.mdn_last_error()

    refused("1..8192", width=0)
    refused("1..8192", width=8193)
    refused("x_dtype", x_dtype=1)
    refused("x_dtype", y_dtype=2)
    refused("gate_kind", gate_kind=4)
    refused("gate_dtype", gate_dtype=1)
    refused("inner_count", inner_count=0)
    refused("null weights", w_pre=None)
    refused("null rows", x=sequence._NormRows())
    refused("null rows", h=sequence._NormRows())
    assert lib.mdn_op_block_norm_forward(None, None) == -1
    empty = sequence._BlockNorm.from_buffer_copy(good)
    empty.rows = 0
    assert lib.mdn_op_block_norm_forward(ctypes.byref(empty), None) == 0
    grad = sequence._BlockNormGrad()
    assert lib.mdn_op_block_norm_backward(ctypes.byref(good), ctypes.byref(grad), None, 0, None) == -1
    for name in ("d_s", "d_h", "d_x", "d_y", "d_gate"):
        getattr(grad, name).data = some
    grad.d_w_post = grad.d_w_pre = some
    assert lib.mdn_op_block_norm_backward(ctypes.byref(good), ctypes.byref(grad), None, 0, None) == -1
    assert "workspace is too small" in lib.mdn_last_error().decode()


@gpu
@pytest.mark.parametrize("width", [24, 64, 181, 300, 2100])
def test_an_infinite_gradient_in_the_last_row(width):
    """It reaches its row and its columns' sums as an infinity, also where lanes past the last row repeat its loads."""
    from mdnav import sequence
    x, _, _ = inputs((5, width), "channel", F32, F32, seed=6)
    leaves = {name: t.requires_grad_() for name, t in x.items()}
    s, h = sequence.block_norm(**leaves)
    d_s, d_h = torch.full_like(s, 0.5), torch.full_like(h, 0.25)
    d_s[4, 3] = float("inf")
    got = torch.autograd.grad([s, h], list(leaves.values()), [d_s, d_h])
    with np.errstate(all="ignore"):
        want = gradients(**host(x), d_s=d_s.double().cpu().numpy(), d_h=d_h.double().cpu().numpy())
    for name, grad in zip(leaves, got):
        a, b = grad.double().cpu().numpy(), want[name]
        assert np.array_equal(np.isnan(a), np.isnan(b)) and np.array_equal(np.isinf(a), np.isinf(b)), name
        assert np.array_equal(np.sign(a[np.isinf(a)]), np.sign(b[np.isinf(b)])), name
