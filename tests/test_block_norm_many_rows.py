"""The norm block over more rows than the GPU has workgroups and lanes for: a workgroup loads its next row while it works
on one, and adds up the rows' shares of the column sums.  Against the formula in float64.

Tolerances as in test_block_norm.py for rows.  A column sum adds R rows in a lane, one after the other: with terms of
random signs a running sum of i terms has grown as sqrt(i), and so has its rounding, sqrt(R) 2^-24 of the sum in all.
4e-6 were taken there for up to 64 rows; here 4e-6 sqrt(R / 64) where there are more."""
import pytest
import torch  # before the library: one HIP runtime in the process

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
TYPES = {"f32": (F32, F32), "bf16": (BF16, BF16), "mixed": (F32, BF16)}
# a few turns of narrow rows (sixteenth, eighth and quarter of a workgroup each), wide rows of one, two and four pieces a lane
SHAPES = [(40001, 64), (20003, 181), (30001, 100), (2101, 1000), (1301, 5120), (1103, 8192), (20011, 2048), (3, 7001, 24)]


def made(shape, kind, x_type, y_type, seed):
    gen = torch.Generator(device="cuda").manual_seed(seed)

    def randn(*s):
        return torch.randn(*s, generator=gen, device="cuda")

    width = shape[-1]
    gate = dict(none=None, channel=(width,), row=(*shape[:-1], 1), element=shape)[kind]
    x = dict(x=randn(*shape).to(x_type), y=(0.5 * randn(*shape) + 0.1).to(y_type), w_post=1 + 0.1 * randn(width),
             w_pre=1 + 0.1 * randn(width), residual_scale=None if kind == "none" else 1 + 0.1 * randn(width),
             gate=None if gate is None else torch.sigmoid(randn(*gate)).to(F32 if kind == "channel" else y_type))
    return x, randn(*shape).to(x_type), randn(*shape).to(y_type)


def formula(x, y, w_post, w_pre, gate, residual_scale, d_s, d_h, eps=1e-6):
    """(s, h, gradients) in float64, by the chain rule."""
    x, y, w_post, w_pre, d_s, d_h = (t.detach().double() for t in (x, y, w_post, w_pre, d_s, d_h))
    g = 1.0 if gate is None else gate.detach().double()
    r = 1.0 if residual_scale is None else residual_scale.detach().double()
    ry = (y.square().mean(-1, keepdim=True) + eps).rsqrt()
    n = y * ry
    s = r * x + g * n * w_post
    rs = (s.square().mean(-1, keepdim=True) + eps).rsqrt()
    h = s * rs * w_pre
    z = d_h * w_pre
    t = d_s + rs * z - s * rs ** 3 * (z * s).mean(-1, keepdim=True)
    d_n = t * g * w_post
    lead = tuple(range(x.dim() - 1))
    d = dict(x=t * r, y=ry * d_n - y * ry ** 3 * (d_n * y).mean(-1, keepdim=True), w_post=(t * g * n).sum(lead),
             w_pre=(d_h * s * rs).sum(lead))
    if residual_scale is not None:
        d["residual_scale"] = (t * x).sum(lead)
    if gate is not None:
        whole = t * n * w_post
        d["gate"] = whole.sum(lead) if gate.dim() == 1 else whole if gate.shape == x.shape else whole.sum(-1, keepdim=True)
    return s, h, d


def near(name, got, want, room):
    low = got.dtype == BF16
    got = got.detach().double()
    assert got.shape == want.shape and bool(torch.isfinite(got).all()), name
    rms = want.square().mean().sqrt()
    err = ((got - want).abs() - (2.0 ** -8 * want.abs() if low else 0.0)).clamp_(min=0.0)
    over = err.square().mean().sqrt()
    assert over <= room * rms, (name, float(over / rms))
    assert bool((err <= 40 * room * torch.maximum(rms, want.abs())).all()), name


@gpu
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("kind", ["none", "channel", "row", "element"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_every_row_of_many(shape, kind, types):
    from mdnav import sequence
    print("case: many rows", shape, kind, types, flush=True)
    x, d_s, d_h = made(shape, kind, *TYPES[types], seed=sum(shape))
    want_s, want_h, want = formula(**x, d_s=d_s, d_h=d_h)
    leaves = {n: t.requires_grad_() for n, t in x.items() if t is not None}
    s, h = sequence.block_norm(**x)
    near("s", s, want_s, 1e-6)
    near("h", h, want_h, 1e-6)
    got = torch.autograd.grad([s, h], list(leaves.values()), [d_s, d_h])
    rows = s.numel() // shape[-1]
    in_a_lane = max(64.0, rows / 256)  # at least 256 workgroups
    for (n, leaf), grad in zip(leaves.items(), got):
        column = n.startswith("w") or n == "residual_scale" or (n, kind) == ("gate", "channel")
        near("d_" + n, grad, want[n], 4e-6 * (in_a_lane / 64) ** 0.5 if column else 1e-6)


@gpu
@pytest.mark.parametrize("types", list(TYPES))
@pytest.mark.parametrize("shape,gate", [((50, 1), (1,)), ((3, 40, 1), (3, 40, 1)), ((70, 1), (70, 1)), ((1,), (1,))], ids=str)
def test_gates_of_one_channel(shape, gate, types):
    """In rows of one element a gate of [1] is the channel's (the row's, where there is one row and no axis), one of
    [..., 1] the row's."""
    from mdnav import sequence
    gen = torch.Generator(device="cuda").manual_seed(1)

    def randn(*s):
        return torch.randn(*s, generator=gen, device="cuda")

    x_type, y_type = TYPES[types]
    x = dict(x=randn(*shape).to(x_type), y=randn(*shape).to(y_type), w_post=randn(1), w_pre=randn(1), gate=randn(*gate), residual_scale=randn(1))
    d_s, d_h = randn(*shape).to(x_type), randn(*shape).to(y_type)
    as_rows = {n: t.reshape(-1, 1) if n in ("x", "y") or (n == "gate" and gate == shape) else t for n, t in x.items()}
    want_s, want_h, want = formula(**as_rows, d_s=d_s.reshape(-1, 1), d_h=d_h.reshape(-1, 1))
    leaves = {n: t.requires_grad_() for n, t in x.items()}
    s, h = sequence.block_norm(**x)
    near("s", s, want_s.reshape(shape), 1e-6)
    near("h", h, want_h.reshape(shape), 1e-6)
    got = torch.autograd.grad([s, h], list(leaves.values()), [d_s, d_h])
    for (n, leaf), grad in zip(leaves.items(), got):
        assert grad.shape == leaf.shape and grad.dtype == leaf.dtype
        # a row of one element leaves of a gradient the share of epsilon: 1e-6 of terms that are larger by a million
        near("d_" + n, grad, want[n].reshape(leaf.shape), 4e-6)


@gpu
@pytest.mark.parametrize("kind", ["none", "channel", "row", "element"])
def test_a_result_that_nothing_asks_for_has_no_share(kind):
    """With one result unused its gradient counts as zeros: what only it depends on gets none, or zeros."""
    from mdnav import sequence
    x, d_s, d_h = made((37, 70), kind, F32, F32, seed=3)
    for which in (0, 1):
        leaves = {n: t.detach().requires_grad_() for n, t in x.items() if t is not None}
        out = sequence.block_norm(**{n: leaves.get(n) for n in x})
        got = dict(zip(leaves, torch.autograd.grad(out[which], list(leaves.values()), (d_s, d_h)[which], allow_unused=True)))
        zero = torch.zeros_like(d_s)
        want = formula(**x, d_s=(d_s, zero)[which], d_h=(zero, d_h)[which])[2]
        for n, grad in got.items():
            if bool(want[n].any()):
                near("d_" + n, grad, want[n], 4e-6)
            else:
                assert grad is None or not bool(grad.any()), n
        assert which == 1 or got["w_pre"] is None or not bool(got["w_pre"].any())
