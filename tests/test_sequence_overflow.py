"""The gated delta rule where finite inputs outgrow fp32: an infinity that arises inside a rollout reaches later
ticks of its episode (in reverse, earlier ones) and nothing else.

The definition is taken in float64, where the same numbers stay finite; ticks that fp32 has left are not compared, all
others are, tick by tick in their own norm.  Tolerances as in test_sequence_ops.py, whose bounds hold for every row."""
import numpy as np
import pytest
import torch  # before the library: one HIP runtime in the process

from test_sequence_ops import NORM, TORCH, host, inputs, rule, rule_gradients

gpu = pytest.mark.gpu

SHAPES = [(70, 6, 1, 1, 64, 64), (64, 6, 1, 2, 128, 128), (90, 6, 1, 1, 40, 72), (50, 6, 2, 4, 16, 9),
          (1200, 6, 1, 1, 64, 64), (1200, 6, 1, 1, 24, 100)]
GROWS, FLAG = 8, 20  # ticks of a rollout, past `first` below


def growing(shape, dtype):
    """A rollout whose envs leave fp32 between ticks `first + GROWS` and `first + FLAG`, where an episode begins:
    (inputs, d_o, first)."""
    t, n, hq, h, kd, vd = shape
    x = host(inputs(*shape, dtype, seed=21, resets=0, gates=dtype))
    first = 480 if t > 1000 else 0  # in a chunk of its own among many, or the first
    grow = slice(first + GROWS, first + FLAG)
    reset = np.zeros((t, n), np.uint8)
    reset[first + FLAG] = 1
    if t > 1000:  # the same start in the segments' middle
        reset[first] = 1
    x["reset"] = reset
    # each tick multiplies the state by 1 - 1e4 along its key
    x["k"][grow, 0] = np.sqrt(1e4 / kd)
    x["beta"][grow, 0] = 1.0
    x["g"][grow, 0] = 0.0
    # decays that are growths, e^144 in all
    x["g"][grow, 1] = 12.0
    # a state of 1e30 and then, in another episode of the chunk, a query of 1e10
    x["v"][first + 2, 2] *= 1e30
    x["q"][first + FLAG + 5, 2] *= 1e10
    # keys of 1e10 with strengths that keep the state small, and a query of 1e30 in the next episode
    x["k"][grow, 3] *= 1e10
    x["beta"][grow, 3] = 1e-25
    x["q"][first + FLAG + 5, 3] *= 1e30
    # the same state as in env 2 beside a gradient of 1e10
    x["v"][first + 2, 4] *= 1e30
    d_o = np.random.default_rng(3).normal(size=(t, n, h, vd))
    d_o[first + FLAG + 5, 4] *= 1e10
    dt = TORCH[dtype]
    out = {name: torch.from_numpy(a).to(torch.float32 if name == "state" else dt if a.dtype != np.uint8 else torch.uint8).cuda()
           for name, a in x.items()}
    return out, torch.from_numpy(d_o).to(dt).cuda(), first


def groups_near(name, got, want, env, groups, dtype):
    """Each group of ticks in its own norm; a single row's share of the errors is at most four times the norm's."""
    low = got.dtype == torch.bfloat16
    got = got.detach().double().cpu().numpy()
    for ticks in groups:
        a, b = got[ticks, env], want[ticks, env]
        assert np.isfinite(a).all(), (name, env, ticks)
        err = np.maximum(np.abs(a - b) - (2.0 ** -8 * np.abs(b) if low else 0.0), 0.0)
        assert np.linalg.norm(err) <= 4 * NORM[dtype] * np.linalg.norm(b), (name, env, ticks, np.linalg.norm(err) / np.linalg.norm(b))


def each(*spans):
    return [slice(i, i + 1) for a, b in spans for i in range(a, b)]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
@pytest.mark.parametrize("final", [True, False], ids=["final", "rows"])
def test_values_that_outgrow_fp32_stay_in_their_episode(shape, dtype, final):
    from mdnav import sequence
    print("case: overflow", shape, dtype, flush=True)
    x, _, first = growing(shape, dtype)
    want_o, want_s = rule(**host(x))
    o, last = sequence.delta_rule(**x, final_state=final)
    t = shape[0]
    for env in range(6):
        spans = [(0, first + GROWS + 1), (first + FLAG, t)] if env < 2 else [(0, t)]
        groups_near("o", o, want_o, env, each(*spans), dtype)
        if final:
            groups_near("state", last[None], want_s[None], env, each((0, 1)), dtype)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients_that_outgrow_fp32_stay_in_their_episode(shape, dtype):
    from mdnav import sequence
    print("case: overflow gradients", shape, dtype, flush=True)
    x, d_o, first = growing(shape, dtype)
    leaves = {name: x[name].requires_grad_() for name in ("q", "k", "v", "g", "beta", "state")}
    o, _ = sequence.delta_rule(**x)
    got = dict(zip(leaves, torch.autograd.grad([o], list(leaves.values()), [d_o])))
    want = rule_gradients(**host(x), d_o=d_o.double().cpu().numpy(), d_state=None)
    t, turn = shape[0], first + FLAG + 6  # past the tick with the large query or gradient
    for env in range(6):
        spans = [(first + FLAG, turn), (turn, t)] + ([(0, first)] if first else [])
        if env >= 4:
            spans += [(first, first + 2), (first + 2, first + FLAG)]
        # a group's norm, as a row can be a small difference of its neighbours: in one here (env 3, the flagged tick
        # of the 40 x 72 heads) the definition itself, in fp32, is 3.8e-5 of the row's own norm away
        for name in ("q", "k", "v", "g", "beta"):
            groups_near("d_" + name, got[name], want[name], env, [slice(*s) for s in spans], dtype)
        if first or env >= 4:
            groups_near("d_state", got["state"][None], want["state"][None], env, each((0, 1)), dtype)
