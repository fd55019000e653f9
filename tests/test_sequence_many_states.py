"""The gated delta rule over more states than the GPU holds workgroups for: each goes through several, and loads the next
one's rows, gates and state while it ends this one.  Against the definition in float64, every state and every gradient.
Tolerances as in test_sequence_ops.py: a state's errors do not depend on its neighbours."""
import pytest
import torch  # before the library: one HIP runtime in the process

from test_sequence_ops import NORM, TORCH, inputs

gpu = pytest.mark.gpu
# up to 1,280 workgroups of narrow heads and 512 of wide ones are on 256 compute units at once, half in the backward pass
SHAPES = [(33, 3001, 1, 1, 64, 64), (70, 1501, 1, 2, 40, 72), (40, 3001, 1, 1, 16, 16), (35, 701, 1, 2, 128, 128),
          (65, 457, 2, 6, 24, 96)]


def definition(x, d_o, d_state=None):
    """(o, last state, gradients) in float64 on the GPU, by elementwise products and sums."""
    t, n, hq, kd = x["q"].shape
    h = x["v"].shape[2]
    q, k = (x[name].double().repeat_interleave(h // hq, 2) for name in ("q", "k"))
    v, g, beta, s = (x[name].double() for name in ("v", "g", "beta", "state"))
    keep = (x["reset"] == 0)[:, :, None, None, None]
    none = torch.zeros((), dtype=torch.float64, device="cuda")
    scale = kd ** -0.5
    before, errors, out = [], [], []
    for i in range(t):
        s = torch.where(keep[i], s, none) * torch.exp(g[i])[..., None, None]
        before.append(s)
        errors.append(v[i] - (s * k[i][..., None]).sum(-2))
        s = s + k[i][..., None] * (beta[i][..., None] * errors[-1])[..., None, :]
        out.append(scale * (s * q[i][..., None]).sum(-2))
    last, after = s, s
    d = {name: torch.zeros_like(y) for name, y in (("q", q), ("k", k), ("v", v), ("g", g), ("beta", beta))}
    grad = torch.zeros_like(s) if d_state is None else d_state.double()
    d_o = d_o.double()
    for i in reversed(range(t)):
        s, u = before[i], beta[i][..., None] * errors[i]
        after = s + k[i][..., None] * u[..., None, :]
        d["q"][i] = scale * (after * d_o[i][..., None, :]).sum(-1)
        grad = grad + scale * q[i][..., None] * d_o[i][..., None, :]
        du = (grad * k[i][..., None]).sum(-2)
        d["beta"][i] = (du * errors[i]).sum(-1)
        dv = beta[i][..., None] * du
        d["v"][i] = dv
        d["k"][i] = (grad * u[..., None, :]).sum(-1) - (s * dv[..., None, :]).sum(-1)
        grad = grad - k[i][..., None] * dv[..., None, :]
        d["g"][i] = torch.where(keep[i][..., 0, 0], (grad * s).sum((-1, -2)), none)
        grad = torch.where(keep[i], grad * torch.exp(g[i])[..., None, None], none)
    for name in ("q", "k"):
        d[name] = d[name].unflatten(2, (hq, h // hq)).sum(3)
    d["state"] = grad
    return torch.stack(out), last, d


def near(name, got, want, dtype, env):
    """By the norm and value by value, as in test_sequence_ops.py, where the definition is finite; and not finite where
    it is not.  `env`: the envs' axis, each of which is looked at by itself too."""
    low = got.dtype == torch.bfloat16
    got = got.detach().double()
    finite = torch.isfinite(want)
    assert torch.equal(finite, torch.isfinite(got)), (name, int((finite != torch.isfinite(got)).sum()))
    want, got = (torch.where(finite, y, torch.zeros_like(y)) for y in (want, got))
    err = (got - want).abs() - (2.0 ** -8 * want.abs() if low else 0.0)
    err = err.clamp_(min=0.0)
    rms = want.square().mean().sqrt()
    assert err.square().mean().sqrt() <= NORM[dtype] * rms, (name, float(err.square().mean().sqrt() / rms))
    assert bool((err <= 40 * NORM[dtype] * torch.maximum(rms, want.abs())).all()), name
    each = err.movedim(env, 0).flatten(1).square().mean(1).sqrt()
    assert bool((each <= 8 * NORM[dtype] * rms).all()), (name, float(each.max() / rms))


def poison(x, d_o):
    """Infinities and NaN in every fifth env, with episodes that begin after them, so that chunks taken tick by tick
    come before and after ordinary ones in the same workgroup."""
    t, n = x["reset"].shape
    for e in range(0, n, 5):
        x["reset"][:, e] = 0
        x["reset"][t // 2, e] = 1
    x["v"][t // 4, 0::20, 0, 0] = float("nan")
    x["k"][t - 2, 5::20, 0, 1] = float("inf")
    x["beta"][t // 4, 10::20] = float("nan")
    x["state"][15::20, :, 0, 0] = float("inf")
    d_o[t // 4, 15::20, 0, 1] = float("nan")


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("poisoned", [False, True], ids=["finite", "poisoned"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_every_state_of_many(shape, poisoned, dtype):
    from mdnav import sequence
    print("case: many states", shape, dtype, "poisoned" if poisoned else "", flush=True)
    x = inputs(*shape, dtype, seed=41 + sum(shape), gates="f32" if shape[3] % 2 else dtype, resets=0.04)
    gen = torch.Generator().manual_seed(5)
    d_o = torch.randn(x["v"].shape, generator=gen).to(TORCH[dtype]).cuda()
    d_s = torch.randn(x["state"].shape, generator=gen).cuda()
    if poisoned:
        poison(x, d_o)
    want_o, want_s, want = definition(x, d_o, d_s)
    leaves = {name: x[name].requires_grad_() for name in ("q", "k", "v", "g", "beta", "state")}
    o, last = sequence.delta_rule(**x, final_state=True)
    near("o", o, want_o, dtype, 1)
    near("state", last, want_s, dtype, 0)
    got = torch.autograd.grad([o, last], list(leaves.values()), [d_o, d_s])
    for (name, leaf), grad in zip(leaves.items(), got):
        near("d_" + name, grad, want[name], dtype, 0 if name == "state" else 1)
    with torch.no_grad():
        near("o by itself", sequence.delta_rule(**x)[0], want_o, dtype, 1)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(5, 8192, 1, 2, 64, 64), (1, 9001, 1, 3, 40, 72)], ids=str)
def test_ticks_of_many_states(shape, dtype):
    from mdnav import sequence
    print("case: ticks of many states", shape, dtype, flush=True)
    x = inputs(*shape, dtype, seed=sum(shape), gates=dtype)
    want_o, want_s, _ = definition(x, torch.zeros_like(x["v"]))
    state = x["state"].clone()
    o = torch.stack([sequence.delta_rule_step(*(x[name][i] for name in ("q", "k", "v", "g", "beta")), state, reset=x["reset"][i])
                     for i in range(shape[0])])
    near("o", o, want_o, dtype, 1)
    near("state", state, want_s, "f32", 0)


@gpu
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("shape", [(4 * 32 * 24 + 5, 120, 1, 1, 64, 64), (4 * 32 * 100 + 5, 4, 1, 1, 128, 128)], ids=str)
def test_many_segments(shape, dtype):
    """Of many states, and a hundred of each of a few, whose maps and gradients ahead of them are more than the GPU
    holds workgroups for."""
    from mdnav import sequence
    print("case: many segments", shape, dtype, flush=True)
    t, n, _, h, kd, vd = shape
    gen = torch.Generator(device="cuda").manual_seed(7)

    def randn(*s):
        return torch.randn(*s, generator=gen, device="cuda")

    dt = TORCH[dtype]
    unit = torch.nn.functional.normalize
    x = dict(q=unit(randn(t, n, 1, kd), dim=-1).to(dt), k=unit(randn(t, n, 1, kd) + randn(1, n, 1, kd), dim=-1).to(dt),
             v=randn(t, n, h, vd).to(dt), g=-torch.exp(1.5 * randn(t, n, h) - 5), beta=torch.sigmoid(randn(t, n, h)),
             state=0.3 * randn(n, h, kd, vd), reset=(torch.rand(t, n, generator=gen, device="cuda") < 0.002).to(torch.uint8))
    d_o, d_s = randn(t, n, h, vd).to(dt), randn(n, h, kd, vd)
    want_o, want_s, want = definition(x, d_o, d_s)
    leaves = {name: x[name].requires_grad_() for name in ("q", "k", "v", "g", "beta", "state")}
    o, last = sequence.delta_rule(**x, final_state=True)
    near("o", o, want_o, dtype, 1)
    near("state", last, want_s, dtype, 0)
    got = torch.autograd.grad([o, last], list(leaves.values()), [d_o, d_s])
    for (name, leaf), grad in zip(leaves.items(), got):
        near("d_" + name, grad, want[name], dtype, 0 if name == "state" else 1)
