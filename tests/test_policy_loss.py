"""The clipped loss over discrete choices (mdnav.policy.clipped_loss, log_prob) against its formula in float64.

Tolerances, set before the first run.  u = 2^-24.  A row's sum of exponentials is off by 2 u for each (hardware's
2^y), u times the mean of |y| (at most the logarithm of the choices and a little, 20) for its argument, and u for each
addition that a term passes, at most 64 and 20 of a tree: 130 u at worst, of which random signs leave a tenth, taken as
16 u.  l has that for each head, the entropy as much again; the loss and its means are sums in 64 bits, so a step's
errors average out: 16 u heads of the terms' mean magnitude, and a rounding.  A choice's gradient is a product of its
share, off by 16 u and u |log p|, and a step's slope; taken as 64 u of the tensor's norm.  bfloat16 gradients are
rounded once more, at most 2^-8 of their value."""
import ctypes
import math

import numpy as np
import pytest
import torch  # before the library: one HIP runtime in the process

gpu = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24
NUMBERS = dict(clip=(0.2, 0.3), kl_coef=0.05, entropy_coef=0.01)


def formula(x, clip=(0.2, 0.2), kl_coef=0.0, entropy_coef=0.0):
    """loss, metrics and the logits' gradient, in float64, by the chain rule."""
    z, a = x["logits"].double(), x["actions"].long()
    top = z.max(-1, keepdim=True).values
    p = torch.exp(z - top)
    total = p.sum(-1, keepdim=True)
    p = p / total
    lp = torch.where(p > 0, z - top - torch.log(total), torch.zeros_like(z))
    h = -(p * lp).sum(-1, keepdim=True)
    l = (z - top - torch.log(total)).gather(-1, a[..., None])[..., 0].sum(-1)
    out = dict(log_prob=l, entropy=h[..., 0].sum(-1))
    if "old_log_prob" not in x:
        return out
    adv = x["advantages"].double()
    r = torch.exp(l - x["old_log_prob"].double())
    low, high = 1.0 - clip[0], 1.0 + clip[1]
    inside = r.clamp(low, high)
    gain = torch.minimum(r * adv, inside * adv)
    slope = torch.where(inside * adv < r * adv, torch.zeros_like(r), -adv * r)
    k = torch.zeros_like(l)
    if x.get("ref_log_prob") is not None:
        far = x["ref_log_prob"].double() - l
        k = torch.exp(far) - far - 1.0
        if kl_coef:  # (0 leaves the term out, infinite or not)
            slope = slope + kl_coef * (1.0 - torch.exp(far))
    counts = torch.ones_like(l, dtype=torch.bool) if x.get("mask") is None else x["mask"] != 0
    n = int(counts.sum())
    by = 1.0 / n if n else 0.0
    terms = [-gain, k, out["entropy"], r, (inside != r).double()]
    means = [t[counts].sum() * by for t in terms]
    out["loss"] = means[0] + (kl_coef * means[1] if kl_coef else 0.0) - entropy_coef * means[2]
    out["metrics"] = torch.stack(means)
    out["sizes"] = torch.stack([t[counts].abs().sum() * by for t in terms])
    one = torch.zeros_like(z).scatter_(-1, a[..., None], 1.0)
    g = slope[..., None, None] * (one - p) + entropy_coef * p * (lp + h)
    out["d_logits"] = torch.where(counts[..., None, None], g * by, torch.zeros_like(g))
    return out


def inputs(steps, heads, choices, dtype=F32, ruled_out=0.0, mask=0.1, ref=True, seed=0, device="cuda", scale=1.5):
    gen = torch.Generator().manual_seed(seed)
    steps = steps if isinstance(steps, tuple) else (steps,)
    z = scale * torch.randn(*steps, heads, choices, generator=gen)
    a = torch.randint(choices, (*steps, heads), generator=gen)
    if ruled_out:
        out = torch.rand(z.shape, generator=gen) < ruled_out
        out.scatter_(-1, a[..., None], False)
        z[out] = -math.inf
    z = z.to(dtype)
    l = torch.log_softmax(z.double(), -1).gather(-1, a[..., None])[..., 0].sum(-1).float()
    x = dict(logits=z, actions=a, old_log_prob=l + 0.3 * torch.randn(steps, generator=gen), advantages=torch.randn(steps, generator=gen),
             ref_log_prob=l + 0.4 * torch.randn(steps, generator=gen) if ref else None,
             mask=torch.rand(steps, generator=gen) >= mask if mask else None)
    return {n: None if t is None else t.to(device) for n, t in x.items()}


def run(x, scale=None, **numbers):
    from mdnav import policy
    z = x["logits"].detach().requires_grad_()
    loss, metrics = policy.clipped_loss(**dict(x, logits=z), **numbers)
    grad, = torch.autograd.grad(loss if scale is None else loss * scale, z)
    assert loss.dtype == F32 and loss.shape == () and metrics.shape == (5,) and not metrics.requires_grad
    assert grad.dtype == z.dtype and grad.shape == z.shape
    return loss.detach(), metrics, grad


def check(x, scale=None, **numbers):
    loss, metrics, grad = run(x, scale, **numbers)
    want = formula(x, **dict(dict(clip=(0.2, 0.2)), **numbers))
    heads = x["logits"].shape[-2]
    room = 16 * U * heads + U
    for i, name in enumerate(("gain", "kl", "entropy", "ratio", "outside")):
        err = 0.0 if float(metrics[i]) == float(want["metrics"][i]) else abs(float(metrics[i]) - float(want["metrics"][i]))
        print("  %s: %.2e of %.2e" % (name, err, room * float(want["sizes"][i])), flush=True)
        # K is a difference of parts up to exp(|l_ref - l|) that are off by 16 u heads themselves; the entropy is one of
        # log s and t log 2 / s, and log s, s at least 1 and off by 16 u of itself, is off by 16 u however small it is.
        # (results are fp32: nothing is smaller than 2^-149)
        assert err <= 2.0 ** -149 + (room * float(want["sizes"][i]) + (room if i in (1, 2) else 0.0)) * (i != 4) + U * (i == 4), name
    beta = numbers.get("kl_coef", 0.0)
    parts = float(want["sizes"][0] + (beta * (want["sizes"][1] + 1) if beta else 0.0) + numbers.get("entropy_coef", 0.0) * (want["sizes"][2] + 1))
    assert abs(float(loss) - float(want["loss"])) <= room * parts
    w, g = want["d_logits"] * (1.0 if scale is None else scale), grad.double()
    err = ((g - w).abs() - (2.0 ** -8 * w.abs() if grad.dtype == BF16 else 0.0)).clamp_(min=0)
    rms = w.square().mean().sqrt()
    print("  d_logits: %.2e" % (err.square().mean().sqrt() / rms if rms else 0.0), flush=True)
    assert err.square().mean().sqrt() <= 64 * U * rms and (err <= 640 * U * torch.maximum(rms, w.abs())).all()
    return want


@pytest.mark.parametrize("ref", [False, True])
def test_the_gradient_here_matches_differences(ref):
    x = inputs(12, 2, 4, seed=5, ref=ref, ruled_out=0.2, device="cpu")
    x["logits"] = x["logits"].double()
    x = {n: t.double() if t is not None and t.dtype == F32 else t for n, t in x.items()}
    numbers = dict(NUMBERS, kl_coef=NUMBERS["kl_coef"] * ref)
    want = formula(x, **numbers)["d_logits"]
    for at in np.ndindex(tuple(x["logits"].shape)):
        if torch.isinf(x["logits"][at]):
            assert want[at] == 0
            continue
        values = []
        for step in (1e-6, -1e-6):
            z = x["logits"].clone()
            z[at] += step
            values.append(formula(dict(x, logits=z), **numbers)["loss"])
        # values near 1 over 2e-6 in float64: 2e-10 of rounding, third derivatives up to 100 give 2e-11
        assert abs((values[0] - values[1]) / 2e-6 - want[at]) < 1e-8, at


# (lanes of a row by its words: 4, 8, 16, 32, a wavefront, four words a lane, a workgroup; of both types)
SHAPES = [(1, 1, 1), (7, 1, 2), (100, 4, 33), (1000, 3, 64), (513, 2, 129), (300, 1, 300), (60, 2, 700), (41, 1, 2047),
          (33, 1, 5000), (5, 2, 70001), (9000, 1, 5), (2, 40, 7)]


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_matches_the_formula(shape, dtype):
    from mdnav import policy
    for i, more in enumerate((dict(), dict(ruled_out=0.2, mask=0.0), dict(ref=False, mask=0.5))):
        print("case: clipped loss", shape, dtype, more, flush=True)
        x = inputs(*shape, dtype, seed=sum(shape) + i, **more)
        numbers = dict(NUMBERS) if x["ref_log_prob"] is not None else dict(clip=0.2, entropy_coef=0.02)
        want = check(x, scale=None if i else -3.0, **dict(numbers, clip=numbers["clip"] if i < 2 else (0.2, 0.2)))
        l, h = policy.log_prob(x["logits"], x["actions"].int() if i else x["actions"])
        heads = shape[1]
        size = torch.maximum(want["log_prob"].abs(), torch.ones_like(want["log_prob"]))
        assert l.dtype == F32 and ((l.double() - want["log_prob"]).abs() <= 130 * U * heads + U * size).all()
        assert ((h.double() - want["entropy"]).abs() <= 400 * U * heads).all()


@gpu
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
@pytest.mark.parametrize("choices", [6, 200, 3000])
def test_which_side_of_the_border(choices, dtype):
    """Ratios that 32-bit sums cannot tell from the border: every step is clipped, or not, as 64 bits say."""
    from mdnav import policy
    steps, low, high = 400, 0.2, 0.25
    x = inputs(steps, 2, choices, dtype, seed=3, mask=0.0, ref=False)
    l = formula(dict(logits=x["logits"], actions=x["actions"]))["log_prob"]
    border = torch.where(torch.arange(steps, device="cuda") % 2 == 0, 1 - low, 1 + high).double()
    x["old_log_prob"] = (l - torch.log(border)).float()  # rounded to one side or the other
    want = formula(x, clip=(low, high))
    r = torch.exp(l - x["old_log_prob"].double())
    assert ((r - border).abs() < 1e-5).all() and 50 < int((r < border).sum()) < 350
    _, metrics, grad = run(x, clip=(low, high))
    clipped = (grad == 0).all(-1).all(-1)
    assert torch.equal(clipped, (want["d_logits"] == 0).all(-1).all(-1)) and 0 < int(clipped.sum()) < steps
    assert abs(float(metrics[4]) - float(want["metrics"][4])) < 1e-7


@gpu
def test_the_first_update():
    """The policy that acted: every ratio is 1, which is inside, also of a clip of nothing where r is exactly 1."""
    from mdnav import policy
    x = inputs(500, 3, 40, seed=8, ref=False)
    x["old_log_prob"], _ = policy.log_prob(x["logits"], x["actions"])
    check(x)
    one = inputs(64, 2, 1, seed=9, ref=False, mask=0.0)  # a single choice: l is 0
    one["old_log_prob"].zero_()
    loss, metrics, grad = run(one, clip=0.0)
    assert float(metrics[3]) == 1.0 and float(metrics[4]) == 0.0 and not grad.any()


@gpu
@pytest.mark.parametrize("choices", [9, 3000])
@pytest.mark.parametrize("dtype", [F32, BF16], ids=["f32", "bf16"])
def test_steps_that_do_not_count(choices, dtype):
    """Whatever they hold, they change nothing and have a gradient of 0; if none counts, all is 0."""
    x = inputs(200, 2, choices, dtype, seed=4, mask=0.3)
    want = run(x, **NUMBERS)
    y = {n: t.clone() for n, t in x.items()}
    off = ~x["mask"]
    y["logits"][off] = float("nan")
    y["logits"][off.nonzero()[0]] = float("inf")
    y["actions"][off] = -100
    for n in ("old_log_prob", "advantages", "ref_log_prob"):
        y[n][off] = float("nan")
    got = run(y, **NUMBERS)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    assert not got[2][off].any()
    for mask in (torch.zeros_like(x["mask"]), torch.zeros_like(x["mask"], dtype=torch.uint8)):
        loss, metrics, grad = run(dict(y, mask=mask), **NUMBERS)
        assert float(loss) == 0 and not metrics.any() and not grad.any()


@gpu
@pytest.mark.parametrize("choices", [5, 64, 3000])
def test_choices_that_are_ruled_out(choices):
    """-inf and the types' lowest values: shares of 0, gradients of 0, and the others as without them."""
    for dtype in (F32, BF16):
        print("case: ruled out", choices, dtype, flush=True)
        x = inputs(50, 2, choices, dtype, seed=6, mask=0.0, scale=1.0)
        wide = {}
        for fill in (-math.inf, torch.finfo(dtype).min):
            z = torch.full((50, 2, choices + 13), fill, dtype=dtype, device="cuda")
            z[..., 7:7 + choices] = x["logits"]
            wide[fill] = run(dict(x, logits=z, actions=x["actions"] + 7), **NUMBERS)
            assert not wide[fill][2][..., :7].any() and not wide[fill][2][..., 7 + choices:].any()
            check(dict(x, logits=z, actions=x["actions"] + 7), **NUMBERS)
        for a, b in zip(*wide.values()):
            assert torch.equal(a, b)
        # a row of lowest values alone is an even choice
        z = torch.full((50, 2, choices), torch.finfo(dtype).min, dtype=dtype, device="cuda")
        check(dict(x, logits=z), **dict(NUMBERS, kl_coef=0.0))
        # very different logits
        check(dict(x, logits=x["logits"] * 1000), **dict(NUMBERS, kl_coef=0.0, clip=(0.2, 0.2)))


@gpu
@pytest.mark.parametrize("choices", [5, 3000])
def test_what_is_not_a_number_shows(choices):
    """A NaN logit, an infinite one, a row with nothing left, an action that is none: NaN in the loss and in that step's
    gradient, the other steps' as they were."""
    x = inputs(60, 2, choices, seed=7, mask=0.0)
    want = run(x, **NUMBERS)[2]
    from mdnav import policy
    for what in ("nan", "inf", "nothing", "past", "negative"):
        print("case: not a number", what, flush=True)
        y = {n: None if t is None else t.clone() for n, t in x.items()}
        if what in ("nan", "inf"):
            y["logits"][3, 1, choices // 2] = float(what)
        elif what == "nothing":
            y["logits"][3, 1] = -math.inf
        else:
            y["actions"][3, 1] = choices if what == "past" else -1
        loss, _, grad = run(y, **NUMBERS)
        l, _ = policy.log_prob(y["logits"], y["actions"])
        keep = torch.arange(60) != 3
        assert torch.isnan(loss) and torch.isnan(l[3]) and torch.isfinite(l[keep]).all()
        assert torch.equal(grad[keep], want[keep]) and torch.isnan(grad[3, 1]).any()


@gpu
def test_layouts():
    """Rows apart, steps in two axes exchanged in memory, integers of 32 bits: the bits of contiguous ones."""
    x = inputs((6, 50), 3, 33, BF16, seed=10)
    want = run(x, **NUMBERS)
    wide = torch.zeros(6, 50, 3, 40, dtype=BF16, device="cuda")
    wide[..., 5:38] = x["logits"]
    heads_first = x["logits"].permute(2, 0, 1, 3).contiguous().permute(1, 2, 0, 3)
    swapped = {n: t.transpose(0, 1).contiguous().transpose(0, 1) for n, t in x.items()}
    for other in (dict(x, logits=wide[..., 5:38]), dict(x, logits=heads_first), swapped, dict(x, actions=x["actions"].int()),
                  dict(x, mask=x["mask"].to(torch.uint8)), dict(x, logits=x["logits"].transpose(2, 3).contiguous().transpose(2, 3))):
        for a, b in zip(run(other, **NUMBERS), want):
            assert torch.equal(a, b)


@gpu
def test_no_steps():
    x = inputs(0, 2, 5, mask=0.0)
    from mdnav import policy
    loss, metrics, grad = run(x, **NUMBERS)
    assert float(loss) == 0 and not metrics.any() and grad.shape == (0, 2, 5)
    assert policy.log_prob(x["logits"], x["actions"])[0].shape == (0,)


@gpu
@pytest.mark.parametrize("shape", [(5000, 3, 20), (70, 1, 9000)], ids=str)
def test_graphs_streams_and_repeats(shape):
    """Two captured graphs, replayed in turn between eager calls, a call on another stream: the same bits."""
    from mdnav import policy
    x = inputs(*shape, seed=11)

    def calls():
        return [*run(x, **NUMBERS), *policy.log_prob(x["logits"], x["actions"])]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graphs = []
    for _ in range(2):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, calls()))
    gen = torch.Generator(device="cuda").manual_seed(1)
    for i in range(4):
        x["logits"].copy_(torch.randn(x["logits"].shape, generator=gen, device="cuda"))
        want = [t.clone() for t in calls()]
        graph, captured = graphs[i % 2]
        graph.replay()
        torch.cuda.synchronize()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            beside = calls()
        torch.cuda.current_stream().wait_stream(side)
        for a, b, c in zip(captured, want, beside):
            assert torch.equal(a, b) and torch.equal(c, b)


@gpu
def test_rows_past_four_gigabytes():
    """Steps 1 MB apart: offsets need more than 32 bits."""
    x = inputs(5000, 2, 20, BF16, seed=12)
    wide = torch.zeros(5000, 524288, dtype=BF16, device="cuda")
    far = wide[:, 1000:1040].unflatten(1, (2, 20))
    far.copy_(x["logits"])
    for a, b in zip(run(dict(x, logits=far), **NUMBERS), run(x, **NUMBERS)):
        assert torch.equal(a, b)


@gpu
def test_what_was_saved_may_move():
    """Saved tensors that a hook brings back elsewhere, or as a view of more, give the same gradient."""
    x = inputs(300, 2, 40, BF16, seed=15)
    loss, want = run(x, **NUMBERS)[0], run(x, **NUMBERS)[-1]
    from mdnav import policy
    for back in (lambda t: t.clone(), lambda t: torch.cat((t, t), -1)[..., :t.shape[-1]]):
        z = x["logits"].clone().requires_grad_()
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t.cpu(), lambda t: back(t.cuda())):
            got = policy.clipped_loss(**dict(x, logits=z), **NUMBERS)[0]
        (g,) = torch.autograd.grad(got, z)
        assert torch.equal(got, loss) and torch.equal(g, want)


@gpu
def test_a_long_row_of_equal_shares():
    """Equal terms round alike in a long sum: 2^-24 for each of a lane's 16 additions, 245 times one of these sums and 10
    joins, 5 more for the exponential and its argument, and half a step of the result, at 15."""
    z = torch.zeros(2, 1, 2000003, device="cuda")
    z[:, 0, 1234567] = 0.2
    actions = torch.tensor([[1234567], [2000002]], device="cuda")
    from mdnav import policy
    l, entropy = policy.log_prob(z, actions)
    want = torch.log_softmax(z.double(), -1)
    room = 276 * U + 2.0 ** -21
    assert (l - want.gather(-1, actions[..., None])[:, 0, 0]).abs().max() < room
    assert (entropy + (want.exp() * want).sum(-1)[:, 0]).abs().max() < 2 * room


# ---------------------------------------------------------------- refusals
def test_refusals(monkeypatch):
    import torch.autograd.forward_ad as forward_ad
    from mdnav import policy
    x = inputs(6, 2, 5, device="cpu")
    with pytest.raises(ValueError, match="not on a GPU"):
        policy.clipped_loss(**x)
    with pytest.raises(ValueError, match="not on a GPU"):
        policy.log_prob(x["logits"], x["actions"])
    monkeypatch.setattr(policy, "_device", lambda names, tensors: torch.device("cpu"))
    for more, error, text in [
            (dict(logits=x["logits"][0, 0]), ValueError, "logits are"), (dict(actions=x["actions"][:, 0]), ValueError, "actions has shape"),
            (dict(logits=x["logits"].double()), TypeError, "logits are"), (dict(actions=x["actions"].float()), TypeError, "actions are"),
            (dict(old_log_prob=x["old_log_prob"][:5]), ValueError, "old_log_prob has shape"),
            (dict(advantages=x["advantages"].double()), TypeError, "advantages is"), (dict(mask=x["mask"].float()), TypeError, "mask is"),
            (dict(ref_log_prob=x["actions"]), ValueError, "ref_log_prob has shape"), (dict(logits=torch.zeros(6, 2, 0)), ValueError, "choices"),
            (dict(clip=-0.1), ValueError, "clip is at least 0"), (dict(clip=float("nan")), ValueError, "clip is at least 0"),
            (dict(kl_coef=0.1, ref_log_prob=None), ValueError, "kl_coef needs"), (dict(actions=None), TypeError, "actions is no tensor"),
            (dict(advantages=x["advantages"].clone().requires_grad_()), TypeError, "advantages is data"),
            (dict(old_log_prob=x["old_log_prob"].clone().requires_grad_()), TypeError, "old_log_prob is data"),
            (dict(entropy_coef=torch.tensor(0.1, requires_grad=True)), TypeError, "entropy_coef is a number")]:
        with pytest.raises(error, match=text):
            policy.clipped_loss(**dict(x, **more))
    with pytest.raises(TypeError, match="logits is data"):
        policy.log_prob(x["logits"].clone().requires_grad_(), x["actions"])
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x["logits"], x["logits"])
        with pytest.raises(NotImplementedError, match="forward-mode"):
            policy.clipped_loss(**dict(x, logits=dual))
        with pytest.raises(NotImplementedError, match="forward-mode"):
            policy.log_prob(dual, x["actions"])


def test_the_c_entries_refuse_before_anything_runs():
    from mdnav import native, policy
    L = native.lib()

    def choices(**more):
        c = policy._Choices()
        for n, v in dict(dict(steps=3, heads=2, choices=5, dtype=0, action_bytes=8, logits=4096, step=10, head=5, actions=4096), **more).items():
            setattr(c, n, v)
        return c

    def loss(**more):
        c = policy._ChoiceLoss()
        for n, v in dict(dict(old_log_prob=4096, advantages=4096, clip_low=0.2, clip_high=0.2, loss=4096, metrics=4096), **more).items():
            setattr(c, n, v)
        return c

    keep, work = ctypes.c_uint64(), ctypes.c_uint64()
    for more, text in [(dict(dtype=2), b"dtype"), (dict(action_bytes=2), b"action_bytes"), (dict(heads=0), b"heads"), (dict(choices=1 << 24), b"choices"),
                       (dict(steps=1 << 50), b"too many"), (dict(logits=None), b"null rows"), (dict(actions=None), b"null rows")]:
        c = choices(**more)
        assert L.mdn_op_choices_log_prob(ctypes.byref(c), 4096, 4096, None) == -1 and text in L.mdn_last_error(), more
        assert L.mdn_op_choices_loss_sizes(ctypes.byref(c), ctypes.byref(keep), ctypes.byref(work)) == -1 and text in L.mdn_last_error(), more
    c = choices()
    assert L.mdn_op_choices_log_prob(ctypes.byref(c), None, 4096, None) == -1
    assert L.mdn_op_choices_loss_sizes(ctypes.byref(c), ctypes.byref(keep), ctypes.byref(work)) == 0
    assert keep.value >= 3 * 2 * 16 + 16 and work.value > 0

    def forward(l, k=4096, kb=keep.value, w=4096, wb=work.value):
        return L.mdn_op_choices_loss_forward(ctypes.byref(c), ctypes.byref(l) if l else None, k, kb, w, wb, None)

    for args, text in [((None,), b"null"), ((loss(old_log_prob=None),), b"null rows"), ((loss(advantages=None),), b"null rows"),
                       ((loss(clip_low=-1.0),), b"clip"), ((loss(clip_high=float("nan")),), b"clip"), ((loss(kl_coef=0.1),), b"ref_log_prob"),
                       ((loss(), None), b"keep"), ((loss(), 4096, keep.value - 1), b"keep"), ((loss(), 4100), b"aligned"),
                       ((loss(), 4096, keep.value, None), b"workspace"), ((loss(), 4096, keep.value, 4096, work.value - 1), b"workspace"),
                       ((loss(), 4096, keep.value, 4100, work.value), b"aligned"), ((loss(loss=None),), b"null results"), ((loss(metrics=None),), b"null results")]:
        assert forward(*args) == -1 and text in L.mdn_last_error(), (args, L.mdn_last_error())
    l = loss()
    for d_loss, d_logits in ((None, 4096), (4096, None)):
        assert L.mdn_op_choices_loss_backward(ctypes.byref(c), ctypes.byref(l), 4096, keep.value, d_loss, d_logits, None) == -1
    assert L.mdn_op_choices_loss_backward(ctypes.byref(c), ctypes.byref(l), 4096, 0, 4096, 4096, None) == -1 and b"keep" in L.mdn_last_error()
