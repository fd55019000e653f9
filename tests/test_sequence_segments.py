"""The gated delta rule where few long states are cut into segments that run side by side: what a segment's map does to
infinities, NaN and zeros is what its ticks would do.  Tolerances as in test_sequence_ops.py."""
import numpy as np
import pytest
import torch  # before the library: one HIP runtime in the process

from test_sequence_ops import TORCH, host, inputs, rule, rule_gradients, same_where_finite

gpu = pytest.mark.gpu
SHAPES = [(1200, 4, 1, 1, 64, 64), (1500, 4, 1, 2, 40, 100), (2100, 4, 1, 1, 128, 128), (1200, 4, 1, 1, 128, 16)]


def fading(shape, dtype):
    """A rollout without flags whose decays leave nothing of a state after a segment: e^-128 and less."""
    x = inputs(*shape, dtype, seed=31, resets=0, gates=dtype)
    x["g"].fill_(-1.0)
    return x


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_nan_outlives_decays(shape, dtype):
    """0 times NaN is NaN: without a flag no decay ends it, in however many segments."""
    from mdnav import sequence
    print("case: fading", shape, dtype, flush=True)
    x = fading(shape, dtype)
    x["state"][0, 0, :, 0] = float("nan")
    x["state"][1, 0, 1, 2] = float("inf")
    x["v"][10, 2, 0, 3] = float("nan")
    with np.errstate(all="ignore"):
        want_o, want_s = rule(**host(x))
    assert np.isnan(want_s[0, 0, :, 0]).all() and np.isnan(want_o[-1, 2, 0, 3])
    o, last = sequence.delta_rule(**x, final_state=True)
    same_where_finite("o", o, want_o, dtype)
    same_where_finite("state", last, want_s, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_nan_outlives_decays_in_reverse(shape, dtype):
    """A gradient of NaN reaches every tick before it, through decays that leave nothing of other gradients."""
    from mdnav import sequence
    print("case: fading gradients", shape, dtype, flush=True)
    x = fading(shape, dtype)
    leaves = {name: x[name].requires_grad_() for name in ("q", "k", "v", "g", "beta", "state")}
    d_o = torch.randn(x["v"].shape, generator=torch.Generator().manual_seed(1)).to(TORCH[dtype]).cuda()
    d_o[shape[0] - 2, 1, 0, 1] = float("nan")
    o, _ = sequence.delta_rule(**x)
    got = torch.autograd.grad([o], list(leaves.values()), [d_o])
    with np.errstate(all="ignore"):
        want = rule_gradients(**host(x), d_o=d_o.double().cpu().numpy(), d_state=None)
    assert np.isnan(want["v"][0, 1, 0, 1]) and np.isfinite(want["v"][:, 0]).all()
    for (name, _), grad in zip(leaves.items(), got):
        same_where_finite("d_" + name, grad, want[name], dtype)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES + [(100, 4, 1, 1, 64, 64), (12, 4, 1, 2, 40, 24)], ids=str)
def test_a_map_that_outgrows_fp32_leaves_zeros_alone(shape, dtype):
    """Keys of length 10 multiply what a state holds by 99 a tick: a segment's map overflows, but columns with
    nothing in them stay empty, and so do their gradients."""
    from mdnav import sequence
    print("case: growing maps", shape, dtype, flush=True)
    t, n, hq, h, kd, vd = shape
    x = inputs(*shape, dtype, seed=32, resets=0, gates=dtype)
    x["k"][:, 1] *= 10.0
    x["beta"][:, 1] = 1.0
    x["g"][:, 1] = 0.0
    for name in ("v", "state"):
        (x[name][:, 1] if name == "v" else x[name][1])[...] = 0.0
    x["v"][t // 2, 1, 0, 5] = 1.0  # one column overflows after this
    leaves = {name: x[name].requires_grad_() for name in ("q", "k", "v", "g", "beta", "state")}
    o, last = sequence.delta_rule(**x, final_state=True)
    others = [c for c in range(vd) if c != 5]
    assert not o[:, 1][..., others].any() and not last[1][..., others].any()
    assert not o[:t // 2, 1].any()
    d_o = torch.randn(x["v"].shape, generator=torch.Generator().manual_seed(2)).to(TORCH[dtype]).cuda()
    d_o[:, 1] = 0.0
    x["v"].data[t // 2, 1, 0, 5] = 0.0
    o, last = sequence.delta_rule(**x)
    assert not o[:, 1].any()
    got = dict(zip(leaves, torch.autograd.grad([o], list(leaves.values()), [d_o])))
    want = rule_gradients(**host(x), d_o=d_o.double().cpu().numpy(), d_state=None)
    for name, grad in got.items():
        here = grad[1] if name == "state" else grad[:, 1]
        assert not here.any(), name
        same_where_finite("d_" + name, grad, want[name], dtype)
