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
        out["g"][i] = np.where(keep[i][:, None] != 0, (grad * before[i]).sum((-1, -2)), 0.0)
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


def same_where_finite(name, got, want, dtype):
    """Infinities and NaN where the definition has them, and near it elsewhere."""
    low = got.dtype == torch.bfloat16
    got = got.detach().double().cpu().numpy()
    bad = ~np.isfinite(want)
    assert np.array_equal(bad, ~np.isfinite(got)), (name, bad.sum(), (~np.isfinite(got)).sum())
    got, want = got[~bad], want[~bad]
    rms = np.sqrt(np.mean(want ** 2))
    err = np.maximum(np.abs(got - want) - (2.0 ** -8 * np.abs(want) if low else 0.0), 0.0)
    assert np.sqrt(np.mean(err ** 2)) <= NORM[dtype] * rms, name


def poisoned(shape, dtype, state=True):
    """A rollout whose envs have infinities and NaN in places, between ticks flagged as an episode's first."""
    t, n, hq, h, kd, vd = shape
    x = inputs(*shape, dtype, seed=11, resets=0, gates=dtype, state=state)
    reset = torch.zeros(t, n, dtype=torch.uint8)
    reset[t // 4], reset[3 * t // 4] = 1, 1
    x["reset"] = reset.cuda()
    half = t // 2
    x["v"][half, 0, 0, 0] = float("nan")     # one column of one state
    x["k"][half, 1, 0, 1] = float("nan")     # a whole state
    x["k"][t // 4 - 1, 2, 0, 0] = float("inf")  # the last tick before a flag
    x["beta"][half, 3] = float("nan")
    x["g"][3 * t // 4 + 1, 4] = float("nan")
    x["q"][half, 5] = float("nan")           # one tick's outputs
    if x["state"] is not None:
        x["state"][6] = float("nan")         # until the first flag
    return x


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(20, 7, 1, 1, 64, 64), (70, 7, 1, 2, 64, 64), (64, 7, 2, 2, 128, 128), (90, 7, 1, 1, 40, 72),
                                   (1200, 7, 1, 1, 64, 64)], ids=str)
def test_infinities_and_nan_stay_where_they_are(shape, dtype):
    """They reach later ticks of their episode and nothing else: no earlier tick, no other episode, env or head."""
    from mdnav import sequence
    print("case: nan", shape, dtype, flush=True)
    x = poisoned(shape, dtype)
    with np.errstate(all="ignore"):
        want_o, want_s = rule(**host(x))
    o, last = sequence.delta_rule(**x, final_state=True)
    same_where_finite("o", o, want_o, dtype)
    same_where_finite("state", last, want_s, dtype)
    o = sequence.delta_rule(**x)[0]
    same_where_finite("o without a final state", o, want_o, dtype)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(20, 7, 1, 1, 64, 64), (70, 7, 1, 2, 64, 64), (64, 7, 2, 2, 128, 128), (90, 7, 1, 1, 40, 72),
                                   (1200, 7, 1, 1, 64, 64)], ids=str)
def test_gradients_of_infinities_and_nan_stay_in_their_episode(shape, dtype):
    from mdnav import sequence
    print("case: nan gradients", shape, dtype, flush=True)
    x = poisoned(shape, dtype)
    leaves = {name: x[name].requires_grad_() for name in ("q", "k", "v", "g", "beta", "state")}
    d_o = torch.randn(x["v"].shape, generator=torch.Generator().manual_seed(1)).to(TORCH[dtype]).cuda()
    d_o[3 * shape[0] // 4 + 2, 0] = float("nan")
    o, _ = sequence.delta_rule(**x)
    got = torch.autograd.grad([o], list(leaves.values()), [d_o])
    with np.errstate(all="ignore"):
        want = rule_gradients(**host(x), d_o=d_o.double().cpu().numpy(), d_state=None)
    for (name, _), grad in zip(leaves.items(), got):
        same_where_finite("d_" + name, grad, want[name], dtype)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decays_of_nothing_and_of_everything(dtype):
    """g = -inf, the type's lowest value and g = 0; beta = 0 and 1; every tick flagged."""
    from mdnav import sequence
    shape = (75, 6, 1, 1, 64, 64)
    x = inputs(*shape, dtype, seed=5, gates=dtype)
    x["g"][10, 0], x["g"][33, 0] = float("-inf"), float("-inf")
    x["g"][:, 1] = torch.finfo(TORCH[dtype]).min
    x["g"][:, 2] = 0.0
    x["beta"][:, 3] = 0.0
    x["beta"][:, 4] = 1.0
    x["reset"][:, 5] = 1
    leaves = {name: x[name].requires_grad_() for name in ("q", "k", "v", "g", "beta", "state")}
    d_o = torch.randn(x["v"].shape, generator=torch.Generator().manual_seed(1)).to(TORCH[dtype]).cuda()
    o, last = sequence.delta_rule(**x, final_state=True)
    got = torch.autograd.grad([o], list(leaves.values()), [d_o])
    want_o, want_s = rule(**host(x))
    near("o", o, want_o, dtype)
    near("state", last, want_s, dtype)
    want = rule_gradients(**host(x), d_o=d_o.double().cpu().numpy(), d_state=None)
    for (name, _), grad in zip(leaves.items(), got):
        near("d_" + name, grad, want[name], dtype)


@gpu
def test_nothing_to_do():
    """No ticks: the state passes through, gradients too; no envs."""
    from mdnav import sequence
    x = inputs(0, 3, 1, 2, 64, 32, "bf16", resets=0)
    x["state"].requires_grad_()
    o, last = sequence.delta_rule(**x, final_state=True)
    assert o.shape == (0, 3, 2, 32) and torch.equal(last, x["state"])
    (d,) = torch.autograd.grad([last], [x["state"]], [torch.ones_like(last)])
    assert torch.equal(d, torch.ones_like(d))
    x = inputs(5, 0, 1, 2, 64, 32, "f32")
    o, last = sequence.delta_rule(**x, final_state=True)
    assert o.shape == (5, 0, 2, 32) and last.shape == (0, 2, 64, 32)
    x = inputs(0, 3, 1, 1, 8, 8, "f32", state=False, resets=0)
    assert not sequence.delta_rule(**x, final_state=True)[1].any()


@gpu
@pytest.mark.parametrize("kd,vd", [(64, 64), (40, 72), (33, 17)])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_strides(kd, vd, dtype):
    """Batch-first rows, heads cut out of wider rows, unaligned rows, broadcast and reversed inputs: the same bits
    as contiguous ones, in results and gradients."""
    from mdnav import sequence
    t, n, h = 45, 3, 2
    x = inputs(t, n, h, h, kd, vd, dtype, gates=dtype)
    gen = torch.Generator().manual_seed(3)
    wide = torch.randn(n, t, h, kd + vd + 5, generator=gen).to(TORCH[dtype]).cuda() * 0.1
    forms = dict(
        batch_first={name: x[name].transpose(0, 1).contiguous().transpose(0, 1) for name in ("q", "k", "v", "g", "beta", "reset")},
        cut=dict(q=wide.transpose(0, 1)[..., 3:3 + kd], k=wide.transpose(0, 1)[..., 1:1 + kd], v=wide.transpose(0, 1)[..., 5:5 + vd]),
        broadcast=dict(v=x["v"][:1].expand(t, n, h, vd), beta=x["beta"][:, :1].expand(t, n, h), g=x["g"][..., :1].expand(t, n, h)),
        heads_inside=dict(q=x["q"].transpose(1, 2).contiguous().transpose(1, 2)),
        columns=dict(q=wide.transpose(0, 1)[..., ::2][..., :kd] if 2 * kd <= kd + vd + 5 else x["q"]),
        booleans=dict(reset=x["reset"].bool()))
    for form, some in forms.items():
        print("case: strides", form, kd, vd, dtype, flush=True)
        y = dict(x, **some)
        z = {name: a.contiguous() for name, a in y.items()}
        z["reset"] = z["reset"].to(torch.uint8)
        d_o = torch.randn(t, n, h, vd, generator=gen).to(TORCH[dtype]).cuda()
        d_turned = d_o.transpose(0, 2).contiguous().transpose(0, 2)
        runs = []
        for args, grad in ((y, d_turned), (z, d_o)):
            leaves = {name: args[name].detach().requires_grad_() for name in ("q", "k", "v", "g", "beta", "state")}
            o, last = sequence.delta_rule(**leaves, reset=args["reset"], final_state=True)
            runs.append([o, last] + list(torch.autograd.grad([o], list(leaves.values()), [grad])))
        assert all(torch.equal(a, b) for a, b in zip(*runs)), form


@gpu
def test_same_bits_every_time():
    from mdnav import sequence
    x = inputs(200, 5, 2, 6, 64, 64, "bf16")
    leaves = [x[name].requires_grad_() for name in ("q", "k", "v", "g", "beta", "state")]
    d_o = torch.randn(x["v"].shape).bfloat16().cuda()
    runs = []
    for _ in range(2):
        o, last = sequence.delta_rule(**x, final_state=True)
        runs.append([o, last] + list(torch.autograd.grad([o], leaves, [d_o])))
    assert all(torch.equal(a, b) for a, b in zip(*runs))


@gpu
def test_on_another_stream():
    """On a side stream, after work of that stream that the inputs come from."""
    from mdnav import sequence
    x = inputs(100, 16, 1, 2, 64, 64, "f32")
    o, last = sequence.delta_rule(**x, final_state=True)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        big = torch.randn(2048, 2048, device="cuda")
        for _ in range(20):
            big = big @ big * 1e-3
        v = x["v"] + 0.0 * big[0, 0]
        o2, last2 = sequence.delta_rule(**dict(x, v=v), final_state=True)
        state = x["state"].clone()
        step = sequence.delta_rule_step(x["q"][0], x["k"][0], v[0], x["g"][0], x["beta"][0], state, reset=x["reset"][0])
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, o2) and torch.equal(last, last2)
    near("step", step, rule(**{n: a[:1] if n != "state" else a for n, a in host(x).items()})[0][0], "f32")


@gpu
def test_a_rollout_in_pieces_is_the_rollout():
    """States carried from piece to piece, and ticks one at a time, end where the rollout ends."""
    from mdnav import sequence
    x = inputs(96, 4, 1, 2, 64, 64, "f32")
    o, last = sequence.delta_rule(**x, final_state=True)
    state, pieces = x["state"], []
    for a, b in ((0, 1), (1, 40), (40, 96)):
        cut = {name: x[name][a:b] for name in ("q", "k", "v", "g", "beta", "reset")}
        piece, state = sequence.delta_rule(**cut, state=state, final_state=True)
        pieces.append(piece)
    near("o", torch.cat(pieces), o.double().cpu().numpy(), "f32")
    near("state", state, last.double().cpu().numpy(), "f32")


@gpu
def test_a_long_cache_of_strides():
    """Rows more than 2^31 elements into their array."""
    from mdnav import sequence
    t, n, h, d = 40, 2, 1, 64
    x = inputs(t, n, h, h, d, d, "bf16")
    apart = (1 << 31) // (t - 1) + 64  # elements between ticks
    room = torch.zeros(t * apart, dtype=torch.bfloat16, device="cuda")
    far = torch.as_strided(room, (t, n, h, d), (apart, d, d, 1))
    far.copy_(x["v"])
    o, last = sequence.delta_rule(**x, final_state=True)
    o2, last2 = sequence.delta_rule(**dict(x, v=far), final_state=True)
    assert torch.equal(o, o2) and torch.equal(last, last2)


def test_refusals_without_a_gpu():
    from mdnav import sequence
    q, g = torch.zeros(2, 3, 1, 8), torch.zeros(2, 3, 1)
    with pytest.raises(ValueError, match="GPU"):
        sequence.delta_rule(q, q, q, g, g)
    with pytest.raises(TypeError, match="no tensor"):
        sequence.delta_rule(None or [1], q, q, g, g)


@gpu
def test_refusals():
    from mdnav import sequence
    q, g = torch.zeros(2, 3, 2, 8).cuda(), torch.zeros(2, 3, 2).cuda()
    v3, g3 = torch.zeros(2, 3, 3, 8).cuda(), torch.zeros(2, 3, 3).cuda()
    big = torch.zeros(2, 3, 2, 129).cuda()
    state = torch.zeros(3, 2, 8, 8).cuda()
    for bad, error, match in (
            (lambda: sequence.delta_rule(q[0], q[0], q[0], g[0], g[0]), ValueError, "ticks"),
            (lambda: sequence.delta_rule(q, q[:, :2], q, g, g), ValueError, "k has shape"),
            (lambda: sequence.delta_rule(q, q, q[:1], g, g), ValueError, "v has shape"),
            (lambda: sequence.delta_rule(q, q, v3, g3, g3), ValueError, "do not divide"),
            (lambda: sequence.delta_rule(big, big, q, g, g), ValueError, "1..128"),
            (lambda: sequence.delta_rule(q.half(), q.half(), q.half(), g, g), TypeError, "float16"),
            (lambda: sequence.delta_rule(q, q, q.bfloat16(), g, g), TypeError, "one type"),
            (lambda: sequence.delta_rule(q, q, q, g.bfloat16(), g.bfloat16()), TypeError, "g and beta"),
            (lambda: sequence.delta_rule(q, q, q, g, g.double()), TypeError, "g and beta"),
            (lambda: sequence.delta_rule(q, q, q, g, g, state=state[:2]), ValueError, "state has shape"),
            (lambda: sequence.delta_rule(q, q, q, g, g, state=state.double()), TypeError, "state"),
            (lambda: sequence.delta_rule(q, q, q, g, g, reset=g[..., 0]), TypeError, "reset"),
            (lambda: sequence.delta_rule(q, q, q, g, g, reset=torch.zeros(3, 2).bool().cuda()), ValueError, "reset"),
            (lambda: sequence.delta_rule(q, q.cpu(), q, g, g), ValueError, "cpu"),
            (lambda: sequence.delta_rule_step(q[0], q[0], q[0], g[0], g[0], state.transpose(2, 3)), ValueError, "contiguous"),
            (lambda: sequence.delta_rule_step(q[0], q[0], q[0], g[0], g[0], None), ValueError, "contiguous")):
        with pytest.raises(error, match=match):
            bad()


def test_the_c_entries_refuse():
    """What the C entries check themselves, before anything is launched."""
    import ctypes
    from mdnav import native, sequence
    lib = native.lib()
    rule_, sizes = sequence._DeltaRule(4, 2, 1, 2, 64, 64, 1, 1, 0.125), sequence._Sizes()

    def refused(text, **fields):
        c = sequence._DeltaRule.from_buffer_copy(rule_)
        for name, value in fields.items():
            setattr(c, name, value)
        rc = lib.mdn_op_delta_rule_forward(ctypes.byref(c), None, 0, None, 0, None)
        assert rc == -1 and text in lib.mdn_last_error().decode(), (rc, lib.mdn_last_error())

    assert lib.mdn_op_delta_rule_sizes(ctypes.byref(rule_), ctypes.byref(sizes)) == 0
    assert (sizes.keep, sizes.forward_workspace) == (0, 0) and sizes.backward_workspace == 2 * 4 * 2 * 2 * 64 * 4
    rule_.ticks = 65
    assert lib.mdn_op_delta_rule_sizes(ctypes.byref(rule_), ctypes.byref(sizes)) == 0
    assert sizes.keep == 2 * 2 * 2 * 64 * 64 * 4
    refused("null rows")
    refused("dtype", dtype=2)
    refused("gate_dtype", gate_dtype=2)
    refused("1..128", k_dim=0)
    refused("1..128", v_dim=129)
    refused("divide", qk_heads=3)
    refused("divide", heads=0)
    refused("too many states", envs=1 << 31)
    assert lib.mdn_op_delta_rule_forward(None, None, 0, None, 0, None) == -1
    empty = sequence._DeltaRule.from_buffer_copy(rule_)
    empty.envs = 0
    assert lib.mdn_op_delta_rule_forward(ctypes.byref(empty), None, 0, None, 0, None) == 0
    some = ctypes.c_void_p(16)
    for name in ("q", "k", "v", "g", "beta", "o"):
        getattr(rule_, name).data = some
    assert lib.mdn_op_delta_rule_forward(ctypes.byref(rule_), some, 8, None, 0, None) == -1
    assert "keep is too small" in lib.mdn_last_error().decode()
    rule_.ticks, rule_.envs = 5000, 1
    assert lib.mdn_op_delta_rule_forward(ctypes.byref(rule_), None, 0, None, 0, None) == -1
    assert "workspace is too small" in lib.mdn_last_error().decode()
    grad = sequence._DeltaRuleGrad()
    assert lib.mdn_op_delta_rule_backward(ctypes.byref(rule_), ctypes.byref(grad), None, 0, None, 0, None) == -1
    assert "null rows" in lib.mdn_last_error().decode()


@gpu
@pytest.mark.parametrize("shape", [(1, 3, 1, 2, 64, 64), (70, 3, 1, 2, 64, 48), (1500, 2, 1, 1, 64, 64), (2500, 1, 1, 2, 128, 128)], ids=str)
def test_a_state_replaced_in_place(shape):
    """The C entry takes the same buffer for the state before and after, of one tick, in chunks and in segments."""
    from mdnav import sequence
    x = inputs(*shape, "bf16", seed=8, resets=0)
    want_o, want_s = sequence.delta_rule(**x, final_state=True)
    for _ in range(3):
        state = x["state"].clone()
        call = sequence._Call(x["q"], x["k"], x["v"], x["g"], x["beta"], state, x["reset"], None)
        o = call.output()
        call.forward(o, state, False)
        assert torch.equal(o, want_o) and torch.equal(state, want_s)


@gpu
def test_a_tick_in_place_is_seen_by_autograd():
    """A backward pass that would read the state of before the tick raises; a state that wants gradients is refused."""
    from mdnav import sequence
    x = inputs(5, 3, 1, 2, 16, 16, "f32", seed=9)
    x["v"].requires_grad_()
    tick = [x[name][0].detach() for name in ("q", "k", "v", "g", "beta")]
    o, _ = sequence.delta_rule(**x)
    before = x["state"]._version
    sequence.delta_rule_step(*tick, x["state"])
    assert x["state"]._version == before + 1
    with pytest.raises(RuntimeError, match="inplace"):
        o.sum().backward()
    learned = x["state"].clone().requires_grad_()
    with pytest.raises(ValueError, match="gradients"):
        sequence.delta_rule_step(*tick, learned)
    with torch.no_grad():
        sequence.delta_rule_step(*tick, learned)
    assert not torch.equal(learned, x["state"])
