"""A scale of the caller's own reaches every path of the gated delta rule: single ticks, chunks, segments, chunks taken
by the definition, and the gradients of each.  Tolerances as in test_sequence_ops.py."""
import numpy as np
import pytest
import torch  # before the library: one HIP runtime in the process

from test_sequence_ops import TORCH, host, inputs, near, rule, rule_gradients, same_where_finite

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("scale", [0.7, -2.5])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(1, 3, 1, 2, 64, 64), (9, 3, 1, 1, 40, 72), (70, 3, 1, 2, 64, 64), (33, 2, 1, 1, 128, 96),
                                   (700, 2, 1, 1, 64, 64)], ids=str)
def test_a_scale(shape, dtype, scale):
    from mdnav import sequence
    print("case: scale", shape, dtype, scale, flush=True)
    x = inputs(*shape, dtype, seed=51, gates=dtype)
    leaves = {name: x[name].requires_grad_() for name in ("q", "k", "v", "g", "beta", "state")}
    gen = torch.Generator().manual_seed(9)
    d_o = torch.randn(x["v"].shape, generator=gen).to(TORCH[dtype]).cuda()
    o, last = sequence.delta_rule(**x, scale=scale, final_state=True)
    want_o, want_s = rule(**host(x), scale=scale)
    near("o", o, want_o, dtype)
    near("state", last, want_s, dtype)
    got = torch.autograd.grad([o], list(leaves.values()), [d_o])
    want = rule_gradients(**host(x), d_o=d_o.double().cpu().numpy(), d_state=None, scale=scale)
    for (name, _), grad in zip(leaves.items(), got):
        near("d_" + name, grad, want[name], dtype)
    with torch.no_grad():
        state = x["state"].detach().clone()
        step = sequence.delta_rule_step(*(x[name][0] for name in ("q", "k", "v", "g", "beta")), state, reset=x["reset"][0], scale=scale)
    near("step", step, want_o[0], dtype)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(70, 3, 1, 2, 64, 64), (40, 3, 1, 1, 24, 100), (700, 3, 1, 1, 64, 64)], ids=str)
def test_a_scale_beside_nan(shape, dtype):
    """In chunks taken by the definition: NaN before a flag, ordinary numbers after it in the same chunk."""
    from mdnav import sequence
    x = inputs(*shape, dtype, seed=52, resets=0, gates=dtype)
    x["reset"] = torch.zeros(shape[:2], dtype=torch.uint8).cuda()
    x["reset"][8::16] = 1
    x["k"][4::32, 0, 0, 1] = float("nan")
    x["q"][4::32, 1] = float("inf")
    leaves = {name: x[name].requires_grad_() for name in ("q", "k", "v", "g", "beta", "state")}
    d_o = torch.randn(x["v"].shape, generator=torch.Generator().manual_seed(9)).to(TORCH[dtype]).cuda()
    o, last = sequence.delta_rule(**x, scale=0.7, final_state=True)
    with np.errstate(all="ignore"):
        want_o, want_s = rule(**host(x), scale=0.7)
        want = rule_gradients(**host(x), d_o=d_o.double().cpu().numpy(), d_state=None, scale=0.7)
    same_where_finite("o", o, want_o, dtype)
    same_where_finite("state", last, want_s, dtype)
    got = torch.autograd.grad([o], list(leaves.values()), [d_o])
    for (name, _), grad in zip(leaves.items(), got):
        same_where_finite("d_" + name, grad, want[name], dtype)
