"""Activations of the linear layer and the gated block far from 0: values and slopes against their formulas in float64.

Tolerances, set before the first run, u = 2^-24.  Up to here values come as z s(z), s from one or two exponentials, a
reciprocal and a few roundings: 2^-20 of the value, and a bfloat16 result half a step, 2^-8, more.  An exponential's
argument a is itself rounded, up to 4 times, which is 4 u a of the value; a is below 90 where the value is a normal
number.  Where it is not, below 2^-126, the value may be 0, and the least reciprocal that is a normal number, times 90,
may stand in for it: 90 * 2^-126 is below 2^-119."""
import pytest
import torch  # before the library: one HIP runtime in the process
from test_dense import ACTS, BF16, F32, U, call

gpu = pytest.mark.gpu
FAR = [-60.0, -79.0, -84.0, -87.5, -89.0, -95.0, -110.0, -1e3, -1e6, -1e30, -3.38e38, 40.0, 95.0, 1e3, 1e30, 3.38e38]


def allowed(want, dtype):
    return (2.0 ** -20 + 4 * 90 * U + (2.0 ** -8 if dtype == BF16 else 0.0)) * want.abs() + 2.0 ** -119


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("rows", [1, 300])
@pytest.mark.parametrize("act", list(ACTS))
def test_far_from_zero(act, rows, dtype):
    """Values of the forward pass, slopes, and the values that a gated block's backward pass makes again (with `up` 1,
    the gradient of its bias in a call of one row)."""
    print("case: far", act, rows, dtype, flush=True)
    x = torch.tensor(FAR).to(dtype).cuda().expand(rows, 16).contiguous().requires_grad_()
    eye, none = torch.eye(16, dtype=dtype).cuda(), torch.zeros(16, 16, dtype=dtype).cuda()
    one = torch.ones(16, dtype=dtype).cuda().requires_grad_()
    f, g = ACTS[act]
    value, slope = f(x.detach().double()), g(x.detach().double())
    y = call(dict(x=x, w=eye), act)
    d_x, = torch.autograd.grad(y, x, torch.ones_like(y))
    gated = call(dict(x=x, w=eye, w_up=none, b_up=one), act)
    d_gated, again = torch.autograd.grad(gated, [x, one], torch.ones_like(y))
    for name, got, want in (("value", y, value), ("gated value", gated, value), ("slope", d_x, slope), ("gated slope", d_gated, slope),
                            ("value again", again if rows == 1 else None, value[0])):
        if got is None:
            continue
        err = (got.detach().double() - want).abs()
        print("  %s: %s" % (name, (err / allowed(want, dtype)).max().item()), flush=True)
        assert (err <= allowed(want, dtype)).all(), (name, got, want)


@gpu
@pytest.mark.parametrize("rows", [30, 480])
def test_the_tail_of_gelu(rows):
    """Every bfloat16 number from -1 to -13, where z Phi(z) ends: half a step of the result, 2^-8, 2^-13 for the
    approximation of Phi / exp(-z^2 / 2), and 4 u 90 for the exponential's argument and the rest.  The slope
    Phi + z phi passes 0: the same of its parts."""
    z = torch.arange(0xBF80, 0xBF80 + 467).to(torch.int16).view(BF16)
    z = torch.cat((z, torch.full((13,), -2.0, dtype=BF16))).reshape(30, 16).repeat(rows // 30, 1)
    assert z.min() < -13 and z.max() == -1 and (z == -1).any()
    print("case: gelu's tail", rows, flush=True)
    x = z.cuda().requires_grad_()
    y = call(dict(x=x, w=torch.eye(16, dtype=BF16).cuda()), "gelu")
    slope, = torch.autograd.grad(y, x, torch.ones_like(y))
    at = x.detach().double()
    share, density = 0.5 * torch.erfc(-at / 2 ** 0.5), torch.exp(-at * at / 2) / (2 * torch.pi) ** 0.5
    room = 2.0 ** -8 + 2.0 ** -13 + 4 * 90 * U
    for name, got, want, size in (("value", y, at * share, (at * share).abs()), ("slope", slope, share + at * density, share + (at * density).abs())):
        err = (got.detach().double() - want).abs() / size
        print("  %s: %.2e of %.2e" % (name, err.max(), room), flush=True)
        assert (err <= room).all(), name
