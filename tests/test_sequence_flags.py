"""What ends an episode in the gated delta rule: a flag, whatever g its tick has, and a decay of nothing, whatever the
state holds.  Both give the bits that a flag with g = 0 gives, in results and gradients."""
import pytest
import torch  # before the library: one HIP runtime in the process

from test_sequence_ops import TORCH, inputs

gpu = pytest.mark.gpu


@gpu
@pytest.mark.parametrize("how", ["nan", "inf", "low", "-inf"])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(3, 3, 1, 2, 64, 64), (70, 3, 1, 1, 40, 72), (700, 3, 1, 1, 64, 64)], ids=str)
def test_ends_of_episodes(shape, dtype, how):
    from mdnav import sequence
    print("case: ends", shape, dtype, how, flush=True)
    x = inputs(*shape, dtype, seed=61, resets=0, gates=dtype)
    at = torch.zeros(shape[:2], dtype=torch.bool).cuda()
    at[2::17, 0] = True
    at[1::23, 1] = True
    x["state"][0] = float("nan")
    x["g"][at] = 0.0
    x["reset"] = at
    y = dict(x, g=x["g"].clone())
    if how in ("nan", "inf"):
        y["g"][at] = float(how)
    else:
        y["g"][at] = -200.0 if how == "low" else float("-inf")
        y["reset"] = None
    d_o = torch.randn(x["v"].shape, generator=torch.Generator().manual_seed(1)).to(TORCH[dtype]).cuda()
    runs = []
    for z in (x, y):
        leaves = {name: z[name].detach().requires_grad_() for name in ("q", "k", "v", "g", "beta", "state")}
        o, last = sequence.delta_rule(**leaves, reset=z["reset"], final_state=True)
        state, tick = z["state"].clone(), int(at[:, 0].nonzero()[0])
        step = sequence.delta_rule_step(*(z[name][tick] for name in ("q", "k", "v", "g", "beta")), state,
                                        reset=None if z["reset"] is None else z["reset"][tick])
        runs.append([o, last, step, state] + list(torch.autograd.grad([o], list(leaves.values()), [d_o])))
    assert torch.isfinite(runs[0][0][2:, 0]).all() and not runs[0][7][at].any()
    for a, b in zip(*runs):
        assert torch.equal(torch.nan_to_num(a, nan=1e30), torch.nan_to_num(b, nan=1e30))
