"""The gated delta rule (mdnav.sequence) against the definition, tick by tick
in float64.

Tolerances, set before the first run.  A bfloat16 result is rounded once, at
most 2^-8 of its value; what it is rounded from and fp32 results of bfloat16
rows pass through at most eight operands kept as two bfloat16 terms (2^-17
each): 6.1e-5 of the result's norm, taken as 6e-5.  fp32 rows are summed in
fp32 over at most 128 + 32 terms per product and three products in a row, 480
roundings of 2^-24 at worst: 2.9e-5 of the norm, of which random signs leave
less than a fifth; taken as 6e-6."""
import numpy as np
import pytest
import torch  # before the library: one HIP runtime in the process

from mdnav import MdnError

gpu = pytest.mark.gpu
TORCH = {"f32": torch.float32, "bf16": torch.bfloat16}
NORM = {"f32": 6e-6, "bf16": 6e-5}


def rule(q, k, v, g, beta, state=None, reset=None, scale=None):
    """The definition in float64: (o, final state); arguments are numpy arrays."""
    t, n, hq, kd = q.shape
    h, vd = v.shape[2:]
    scale = kd ** -0.5 if scale is None else scale
    q, k = (np.repeat(x.astype(np.float64), h // hq, axis=2) for x in (q, k))
    s = np.zeros((n, h, kd, vd)) if state is None else state.astype(np.float64)
    o = np.zeros((t, n, h, vd))
    for i in range(t):
        if reset is not None:
            s = np.where((reset[i] != 0)[:, None, None, None], 0.0, s)
        s = s * np.exp(g[i].astype(np.float64))[..., None, None]
        u = beta[i].astype(np.float64)[..., None] * (v[i] - np.einsum("nhkv,nhk->nhv", s, k[i]))
        s = s + k[i][..., None] * u[..., None, :]
        o[i] = scale * np.einsum("nhkv,nhk->nhv", s, q[i])
    return o, s


def rule_gradients(q, k, v, g, beta, state, reset, d_o, d_state, scale=None):
    """The definition's gradients in float64, tick by tick in reverse."""
    t, n, hq, kd = q.shape
    h, vd = v.shape[2:]
    shared = h // hq
    scale = kd ** -0.5 if scale is None else scale
    q, k = (np.repeat(x.astype(np.float64), shared, axis=2) for x in (q, k))
    s = np.zeros((n, h, kd, vd)) if state is None else state.astype(np.float64)
    keep = np.ones((t, n)) if reset is None else (reset == 0).astype(np.float64)
    before, after, error = [], [], []
    for i in range(t):
        s = np.where(keep[i][:, None, None, None] != 0, s, 0.0)
        s = s * np.exp(g[i].astype(np.float64))[..., None, None]
        before.append(s)
        error.append(v[i] - np.einsum("nhkv,nhk->nhv", s, k[i]))
        s = s + k[i][..., None] * (beta[i].astype(np.float64)[..., None] * error[-1])[..., None, :]
        after.append(s)
    out = {name: np.zeros(x.shape) for name, x in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta))}
    grad = np.zeros_like(s) if d_state is None else d_state.astype(np.float64)
    for i in reversed(range(t)):
        b = beta[i].astype(np.float64)[..., None]
        out["q"][i] = scale * np.einsum("nhkv,nhv->nhk", after[i], d_o[i])
        grad = grad + scale * q[i][..., None] * d_o[i][..., None, :]
        du = np.einsum("nhkv,nhk->nhv", grad, k[i])
        out["beta"][i] = (du * error[i]).sum(-1)
        out["v"][i] = b * du
        out["k"][i] = np.einsum("nhkv,nhv->nhk", grad, b * error[i]) - np.einsum("nhkv,nhv->nhk", before[i], b * du)
        grad = grad - k[i][..., None] * (b * du)[..., None, :]
        out["g"][i] = (grad * before[i]).sum((-1, -2)) * keep[i][:, None]
        grad = np.where(keep[i][:, None, None, None] != 0, grad * np.exp(g[i].astype(np.float64))[..., None, None], 0.0)
    for name in ("q", "k"):
        out[name] = out[name].reshape(t, n, hq, shared, kd).sum(3)
    out["state"] = grad
    return out


def test_the_gradients_here_match_differences():
    """rule_gradients against central differences of rule(): every input, with
    resets, shared heads and the final state's gradient."""
    rng = np.random.default_rng(3)
    t, n, hq, h, kd, vd = 6, 2, 1, 2, 3, 4
    x = dict(q=rng.normal(size=(t, n, hq, kd)), k=0.6 * rng.normal(size=(t, n, hq, kd)), v=rng.normal(size=(t, n, h, vd)),
             g=-rng.uniform(0.01, 0.5, (t, n, h)), beta=rng.uniform(0.1, 0.9, (t, n, h)),
             state=rng.normal(size=(n, h, kd, vd)))
    reset = np.zeros((t, n), np.uint8)
    reset[2, 0] = reset[4, 1] = 1
    d_o, d_s = rng.normal(size=(t, n, h, vd)), rng.normal(size=(n, h, kd, vd))

    def value(y):
        o, s = rule(y["q"], y["k"], y["v"], y["g"], y["beta"], y["state"], reset)
        return (o * d_o).sum() + (s * d_s).sum()

    grads = rule_gradients(**x, reset=reset, d_o=d_o, d_state=d_s)
    for name, array in x.items():
        for at in np.ndindex(array.shape):
            y = {m: a.copy() for m, a in x.items()}
            y[name][at] += 1e-6
            up = value(y)
            y[name][at] -= 2e-6
            # a difference of values near 10 over 2e-6 in float64: 1e-9 of rounding, 1e-11 of the third derivative
            assert abs((up - value(y)) / 2e-6 - grads[name][at]) < 1e-7, (name, at)


def inputs(t, n, hq, h, kd, vd, dtype, seed=0, resets=0.1, gates="f32", state=True):
    """Device tensors of a rollout; keys of an environment resemble each other."""
    gen = torch.Generator().manual_seed(seed)

    def randn(*shape):
        return torch.randn(*shape, generator=gen)

    def unit(x):
        return x / x.norm(dim=-1, keepdim=True)

    dt, gt = TORCH[dtype], TORCH[gates]
    x = dict(q=unit(randn(t, n, hq, kd)).to(dt), k=unit(randn(t, n, hq, kd) + randn(1, n, hq, kd)).to(dt),
             v=randn(t, n, h, vd).to(dt), g=(-torch.exp(1.5 * randn(t, n, h) - 3)).to(gt),
             beta=torch.sigmoid(randn(t, n, h)).to(gt))
    x["reset"] = (torch.rand(t, n, generator=gen) < resets).to(torch.uint8) if resets else None
    x["state"] = 0.3 * randn(n, h, kd, vd) if state else None
    return {name: None if y is None else y.cuda() for name, y in x.items()}


def host(x):
    return {name: None if y is None else y.detach().float().cpu().numpy() if y.is_floating_point() else y.cpu().numpy()
            for name, y in x.items()}


def near(name, got, want, dtype):
    """A result against float64: by its norm, and, rounded to bfloat16, each value."""
    low = got.dtype == torch.bfloat16
    got = got.detach().double().cpu().numpy()
    assert got.shape == want.shape, name
    assert np.isfinite(got).all(), name
    if not want.size:
        return
    rms = np.sqrt(np.mean(want ** 2))
    err = np.abs(got - want)
    room = 2.0 ** -8 * np.abs(want) if low else 0.0
    over = np.sqrt(np.mean(np.maximum(err - room, 0.0) ** 2))
    print("  %s: norm of the error past its rounding %.2e" % (name, over / rms if rms else over), flush=True)
    assert over <= NORM[dtype] * rms, (name, over / rms)
    # single values: no farther than 40 times the norm's share
    assert np.all(err - room <= 40 * NORM[dtype] * np.maximum(rms, np.abs(want))), name


SHAPES = [
    # ticks, envs, query heads, heads, K, V
    (1, 1, 1, 1, 64, 64),
    (2, 3, 1, 1, 64, 64),
    (31, 2, 2, 2, 64, 64),
    (32, 2, 1, 2, 64, 64),
    (33, 5, 2, 6, 64, 64),
    (64, 1, 1, 1, 128, 128),
    (97, 2, 1, 3, 128, 64),
    (70, 3, 2, 2, 64, 128),
    (40, 2, 1, 1, 1, 1),
    (50, 2, 1, 2, 7, 33),
    (65, 2, 2, 4, 40, 72),
    (130, 1, 1, 1, 127, 101),
    (300, 1, 1, 2, 16, 48),
    # few states of many ticks: segments side by side
    (517, 1, 1, 1, 64, 64),
    (700, 2, 1, 2, 128, 128),
    (1500, 1, 1, 3, 40, 100),
    (2100, 3, 1, 1, 33, 7),
]


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_rollout_matches_the_definition(shape, dtype):
    from mdnav import sequence
    print("case: delta_rule", shape, dtype, flush=True)
    x = inputs(*shape, dtype, seed=sum(shape))
    o, last = sequence.delta_rule(**x, final_state=True)
    assert o.dtype == TORCH[dtype] and last.dtype == torch.float32
    want_o, want_s = rule(**host(x))
    near("o", o, want_o, dtype)
    near("state", last, want_s, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [s for s in SHAPES if s[0] <= 33] + [(5, 7, 1, 4, 128, 128), (4, 3, 2, 2, 100, 5)], ids=str)
def test_ticks_one_at_a_time_match_the_definition(shape, dtype):
    """The fleet's step, tick after tick on one state, against the rollout's definition."""
    from mdnav import sequence
    print("case: delta_rule_step", shape, dtype, flush=True)
    x = inputs(*shape, dtype, seed=1 + sum(shape), gates=dtype)
    state = x["state"].clone()
    rows = []
    for i in range(shape[0]):
        rows.append(sequence.delta_rule_step(x["q"][i], x["k"][i], x["v"][i], x["g"][i], x["beta"][i], state,
                                             reset=x["reset"][i]))
    want_o, want_s = rule(**host(x))
    near("o", torch.stack(rows), want_o, dtype)
    near("state", state, want_s, "f32")


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_gradients_match_the_definition(shape, dtype):
    """Every gradient, the final state's in and the starting state's out; on
    half of the shapes the gates have the rows' type."""
    from mdnav import sequence
    print("case: delta_rule gradients", shape, dtype, flush=True)
    x = inputs(*shape, dtype, seed=2 + sum(shape), gates=dtype if sum(shape) % 2 else "f32")
    leaves = {name: x[name].requires_grad_() for name in ("q", "k", "v", "g", "beta", "state")}
    gen = torch.Generator().manual_seed(9)
    d_o = torch.randn(x["v"].shape, generator=gen).to(TORCH[dtype]).cuda()
    d_s = torch.randn(x["state"].shape, generator=gen).cuda()
    o, last = sequence.delta_rule(**x, final_state=True)
    got = torch.autograd.grad([o, last], list(leaves.values()), [d_o, d_s])
    want = rule_gradients(**host(x), d_o=d_o.double().cpu().numpy(), d_state=d_s.double().cpu().numpy())
    for (name, leaf), grad in zip(leaves.items(), got):
        assert grad.dtype == leaf.dtype
        near("d_" + name, grad, want[name], dtype)
