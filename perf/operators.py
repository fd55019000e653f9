"""Performance cases of the recurrent-policy operators: the memory that a
policy keeps over an episode (the gated delta rule) and the norms around the
block that holds it.

``listed()`` names the cases, ``draw(rng)`` gives further ones of the same
ranges, ``prepare(case, seed)`` makes what a program holds before the call,
``run(state)`` does one pass, ``work(case)`` counts what the pass cannot do
without and ``exact(case, seed)`` is the result in 64 bits.  Where ``own`` is
true the pass calls ``mdnav.sequence``; where it is false it is elementary
tensor code in 32 bits.

The gated delta rule, per environment and head, with a state S of K x V:

    S <- 0 where the tick is flagged as an episode's first
    S <- exp(g) S;  u = beta (v - S^T k);  S <- S + k u^T;  o = scale S^T q

Rows are time-major, [ticks][environments][heads][width], as the rollout
buffers are; several value heads may share one query and key head.

The norm block, per row, around a branch y of a residual stream x:

    s = r x + gate (y / rms(y)) w_post;   h = (s / rms(s)) w_pre

with a residual scale r per channel and a gate per channel, per row or per
element.

The kinds of case:

* ``step``   one tick of every environment: the state is read and replaced;
* ``scan``   whole rollouts forward, from the states the fleet has, to the
             states after it;
* ``train``  the same forward, then every gradient;
* ``norm``   the norm block forward;
* ``norm_train``  the norm block forward, then every gradient.
"""
import math
import os
import sys

import torch

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

own = False

BF16, F32 = "bf16", "f32"


# ---------------------------------------------------------------- the cases
def _delta(name, kind, envs, ticks, qk_heads, heads, k, v, dtype, **more):
    return dict(name=name, kind=kind, envs=envs, ticks=ticks, qk_heads=qk_heads, heads=heads, k=k, v=v, dtype=dtype,
                **more)


def listed():
    return [
        # one tick of the task training fleet, 128 environments, one head of
        # the small policy's 64 units: latency
        _delta("step_task_fleet", "step", 128, 1, 1, 1, 64, 64, F32),
        # one tick of the headline fleet inside a rollout
        _delta("step_headline_fleet", "step", 8192, 1, 4, 4, 64, 64, BF16),
        # an odd fleet with shared query heads and widths off the tile
        _delta("step_ragged_fleet", "step", 3001, 1, 2, 6, 40, 72, BF16),
        # the headline rollout, 8,192 x 128, evaluated forward
        _delta("scan_headline", "scan", 8192, 128, 4, 4, 64, 64, BF16, final=0),
        # two flight logs of 25 minutes at 20 Hz read from the start, to the
        # state that the flight goes on from: few rows, a long axis
        _delta("scan_long_log", "scan", 2, 30011, 4, 8, 128, 128, BF16, final=1),
        # the update on the reference's benchmark rollout, 8,192 x 32
        _delta("train_reference_rollout", "train", 8192, 32, 4, 4, 64, 64, BF16),
        # the capacity policy's width, 5,120 = 40 heads of 128
        _delta("train_capacity_width", "train", 128, 64, 40, 40, 128, 128, BF16),
        # a ragged rollout in 32 bits, shared query heads, odd widths
        _delta("train_ragged_f32", "train", 1000, 37, 2, 6, 40, 72, F32),
        # the block's norms for one tick of the task training fleet: latency
        dict(name="norm_task_fleet", kind="norm", rows=128, width=64, dtype=F32, gate="channel"),
        # an odd width in 32 bits (the actor's 181 inputs), one gate per row
        dict(name="norm_train_ragged", kind="norm_train", rows=37000, width=181, dtype=F32, gate="row"),
        # the reference's benchmark rollout through a block of 256 units
        dict(name="norm_train_rollout", kind="norm_train", rows=8192 * 32, width=256, dtype=BF16, gate="channel"),
        # the capacity policy's width, a gate for each element
        dict(name="norm_train_capacity", kind="norm_train", rows=32768, width=5120, dtype=BF16, gate="element"),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["step", "scan", "train", "train", "norm", "norm_train", "norm_train"])
    dtype = rng.choice([BF16, BF16, F32])
    if kind.startswith("norm"):
        width = _log(rng, 48, 5120)
        rows = min(_log(rng, 1 if kind == "norm" else 100, 1 << 18), (1 << 26) // width)
        return dict(kind=kind, rows=rows, width=width, dtype=dtype, gate=rng.choice(["channel", "row", "element"]))
    shared = rng.choice([1, 1, 2, 3])
    qk_heads = rng.choice([1, 2, 4])
    k, v = rng.choice([(64, 64), (64, 64), (128, 128), (rng.randint(16, 128), rng.randint(16, 128))])
    heads = qk_heads * shared
    case = dict(kind=kind, qk_heads=qk_heads, heads=heads, k=k, v=v, dtype=dtype)
    if kind == "step":
        return dict(case, envs=_log(rng, 1, min(8192, (1 << 27) // (heads * k * v))), ticks=1)
    # states and rows of the largest listed cases bound the rest
    most = (8192 * 32 if kind == "train" else 8192 * 64) * 4 * 64 // (heads * max(k, v))
    if dtype == F32:
        most //= 2
    ticks = rng.choice([rng.randint(1, 40), _log(rng, 24, 256), _log(rng, 24, 256), _log(rng, 256, 8192)])
    envs = _log(rng, 1, max(1, min(8192, most // ticks)))
    if kind == "scan":
        case["final"] = rng.choice([0, 1])
    return dict(case, envs=envs, ticks=ticks)


# ---------------------------------------------------------------- preparation
def _type(case):
    return torch.bfloat16 if case["dtype"] == BF16 else torch.float32


def _unit(x):
    return x / torch.sqrt(x.square().sum(-1, keepdim=True) + 1e-6)


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    kind = case["kind"]
    dt = _type(case)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def rand(*shape):
        return torch.rand(*shape, generator=gen, device="cuda")

    if kind.startswith("norm"):
        rows, width = case["rows"], case["width"]
        gate = {"channel": (width,), "row": (rows, 1), "element": (rows, width)}[case["gate"]]
        st = dict(kind=kind, x=randn(rows, width).to(dt), y=(0.5 * randn(rows, width) + 0.1).to(dt),
                  w_post=1.0 + 0.1 * randn(width), w_pre=1.0 + 0.1 * randn(width),
                  gate=torch.sigmoid(randn(*gate)).to(torch.float32 if case["gate"] == "channel" else dt),
                  residual_scale=1.0 + 0.1 * randn(width), eps=1e-6)
        if kind == "norm_train":
            st["ds"], st["dh"] = randn(rows, width).to(dt), randn(rows, width).to(dt)
            for name in ("x", "y", "w_post", "w_pre", "gate", "residual_scale"):
                st[name].requires_grad_()
        return st

    t, n, hq, h, k, v = (case[x] for x in ("ticks", "envs", "qk_heads", "heads", "k", "v"))
    # keys of one environment resemble each other, as the observations of
    # one flight do; queries and keys are normalised, as the policy does it
    q = _unit(randn(t, n, hq, k)).to(dt)
    key = _unit(randn(t, n, hq, k) + randn(1, n, hq, k)).to(dt)
    val = randn(t, n, h, v).to(dt)
    # per-tick decays from almost none to a half, strengths around a half
    g = (-torch.exp(1.5 * randn(t, n, h) - 3.0)).clamp_(min=-8.0)
    beta = torch.sigmoid(randn(t, n, h))
    # episodes end in 2 % of the ticks
    reset = (rand(t, n) < 0.02).to(torch.uint8)
    start = 0.3 * randn(n, h, k, v)
    if kind == "step":
        return dict(kind=kind, q=q[0], k=key[0], v=val[0], g=g[0].to(dt), beta=beta[0].to(dt), reset=reset[0],
                    state=start)
    st = dict(kind=kind, q=q, k=key, v=val, g=g.to(dt), beta=beta.to(dt), reset=reset, state=start)
    if kind == "scan":
        st["final"] = bool(case["final"])
    else:
        st["do"] = randn(t, n, h, v).to(dt)
        for name in ("q", "k", "v", "g", "beta"):
            st[name].requires_grad_()
        if case["dtype"] == F32:  # in 32 bits the starting state is learned too
            st["state"].requires_grad_()
    return st


# ---------------------------------------------------------------- one pass
def _leaves(st):
    names = [n for n in ("q", "k", "v", "g", "beta", "state", "x", "y", "w_post", "w_pre", "gate", "residual_scale")
             if n in st and st[n].requires_grad]
    return names, [st[n] for n in names]


def _gradients(st, outputs, seeds):
    names, leaves = _leaves(st)
    return dict(zip(["d_" + n for n in names], torch.autograd.grad(outputs, leaves, seeds)))


def run(st):
    if own:
        return _run_own(st)
    kind = st["kind"]
    if kind.startswith("norm"):
        s, h = _plain_norm(st)
        out = dict(s=s.detach(), h=h.detach())
        if kind == "norm_train":
            out.update(_gradients(st, [s, h], [st["ds"], st["dh"]]))
        return out
    if kind == "step":
        o, new = _plain_step(st)
        st["state"] = new
        return dict(o=o, state=new)
    if kind == "scan":
        with torch.no_grad():
            o, last = _plain_scan(st)
        return dict(o=o, state=last) if st["final"] else dict(o=o)
    o, _ = _plain_scan(st)
    return dict(o=o.detach(), **_gradients(st, [o], [st["do"]]))


def _run_own(st):
    if os.path.join(ROOT, "metal-drone-nav_amd") not in sys.path:
        sys.path.insert(0, os.path.join(ROOT, "metal-drone-nav_amd"))
    from mdnav import sequence

    kind = st["kind"]
    if kind.startswith("norm"):
        s, h = sequence.block_norm(st["x"], st["y"], st["w_post"], st["w_pre"], gate=st["gate"],
                                   residual_scale=st["residual_scale"], eps=st["eps"])
        out = dict(s=s.detach(), h=h.detach())
        if kind == "norm_train":
            out.update(_gradients(st, [s, h], [st["ds"], st["dh"]]))
        return out
    if kind == "step":
        o = sequence.delta_rule_step(st["q"], st["k"], st["v"], st["g"], st["beta"], st["state"], reset=st["reset"])
        return dict(o=o, state=st["state"])
    if kind == "scan":
        with torch.no_grad():
            o, last = sequence.delta_rule(st["q"], st["k"], st["v"], st["g"], st["beta"], state=st["state"],
                                          reset=st["reset"], final_state=st["final"])
        return dict(o=o, state=last) if st["final"] else dict(o=o)
    o, _ = sequence.delta_rule(st["q"], st["k"], st["v"], st["g"], st["beta"], state=st["state"], reset=st["reset"])
    return dict(o=o.detach(), **_gradients(st, [o], [st["do"]]))


# ---------------------------------------------------------------- plain forms
def _plain_norm(st):
    dt = st["x"].dtype
    x, y, gate = st["x"].float(), st["y"].float(), st["gate"].float()
    n = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + st["eps"])
    s = st["residual_scale"] * x + gate * (n * st["w_post"])
    h = s * torch.rsqrt(s.square().mean(-1, keepdim=True) + st["eps"]) * st["w_pre"]
    return s.to(dt), h.to(dt)


def _plain_step(st):
    shared = st["v"].shape[1] // st["q"].shape[1]
    q, k = (st[n].float().repeat_interleave(shared, 1) for n in ("q", "k"))
    decay = torch.exp(st["g"].float()) * (st["reset"] == 0)[:, None]
    s = decay[..., None, None] * st["state"]
    u = st["beta"].float()[..., None] * (st["v"].float() - (s * k[..., None]).sum(-2))
    s = s + k[..., None] * u[..., None, :]
    o = (s * q[..., None]).sum(-2) * st["q"].shape[-1] ** -0.5
    return o.to(st["v"].dtype), s


def _unit_lower_inverse(a):
    """(1 + a)^-1 of strictly lower triangular matrices whose size is a power
    of two: the inverses x and y of two neighbouring diagonal blocks join to
    [[x, 0], [-y a' x, y]], for all pairs of blocks at once."""
    c = a.shape[-1]
    i = torch.arange(c, device=a.device)
    inv = torch.eye(c, device=a.device).to(a.dtype).expand_as(a)
    b = 1
    while b < c:
        joined = (i[:, None] // b == i[None, :] // b + 1) & (i[:, None] // b % 2 == 1)
        inv = inv - inv @ (a * joined) @ inv
        b *= 2
    return inv


def _plain_scan(st, chunk=64):
    """The rule in chunks: inside a chunk the u of its ticks solve a unit
    lower triangular system, between chunks the state is carried."""
    t, n, hq, kd = st["q"].shape
    h, vd = st["v"].shape[2:]
    c = min(chunk, 1 << (t - 1).bit_length())
    nc = -(-t // c)

    def rows(x, heads):  # [t][n][heads][...] -> [n][h][nc][c][...], 32 bits, padded with zeros
        x = x.float().repeat_interleave(h // heads, 2)
        x = torch.nn.functional.pad(x, [0, 0] * (x.dim() - 1) + [0, nc * c - t])
        x = x.unflatten(0, (nc, c))
        return x.permute([2, 3, 0, 1] + list(range(4, x.dim())))

    q, k, v = rows(st["q"], hq), rows(st["k"], hq), rows(st["v"], h)
    g, beta = rows(st["g"], h), rows(st["beta"], h)
    first = rows(st["reset"][..., None].expand(t, n, h), h) != 0
    episode = first.cumsum(-1)
    decay = torch.where(first, torch.zeros_like(g), g).cumsum(-1)
    i = torch.arange(c, device=q.device)
    seen = (episode[..., :, None] == episode[..., None, :]) & (i[:, None] >= i[None, :])
    gap = decay[..., :, None] - decay[..., None, :]
    within = torch.where(seen, torch.exp(torch.where(seen, gap, torch.zeros_like(gap))), torch.zeros_like(gap))
    before = torch.where(episode == 0, torch.exp(decay), torch.zeros_like(decay))
    after = within[..., -1, :]
    kt = k.transpose(-1, -2)
    lower = (within * (k @ kt) * beta[..., None]).tril(-1)
    solve = _unit_lower_inverse(lower) * beta[..., None, :]
    uv, uk = solve @ v, (solve * before[..., None, :]) @ k
    scores = within * (q @ kt) * kd ** -0.5
    q = q * (before * kd ** -0.5)[..., None]
    kt = (k * after[..., None]).transpose(-1, -2)
    s, out = st["state"], []
    for j in range(nc):
        u = uv[:, :, j] - uk[:, :, j] @ s
        out.append(q[:, :, j] @ s + scores[:, :, j] @ u)
        s = before[:, :, j, -1, None, None] * s + kt[:, :, j] @ u
    o = torch.stack(out, 2).permute(2, 3, 0, 1, 4).flatten(0, 1)[:t]
    return o.to(st["v"].dtype), s


# ---------------------------------------------------------------- what a pass cannot do without
def work(case):
    size = 2 if case["dtype"] == BF16 else 4
    if case["kind"].startswith("norm"):
        cells = case["rows"] * case["width"]
        gate = {"channel": 4 * case["width"], "row": size * case["rows"], "element": size * cells}[case["gate"]]
        if case["kind"] == "norm":
            return dict(bytes=4 * size * cells + gate + 12 * case["width"], flops=10 * cells)
        return dict(bytes=8 * size * cells + 2 * gate + 24 * case["width"], flops=40 * cells)
    t, n, hq, h, k, v = (case[x] for x in ("ticks", "envs", "qk_heads", "heads", "k", "v"))
    state, qk, val, gates = 4 * n * h * k * v, 2 * size * t * n * hq * k, size * t * n * h * v, t * n * h
    flops = 6 * t * n * h * k * v
    if case["kind"] == "step":
        return dict(bytes=2 * state + qk + 2 * val + 2 * size * gates + n, flops=flops)
    gates *= 2 * size
    if case["kind"] == "scan":
        return dict(bytes=state * (1 + case["final"]) + qk + 2 * val + gates + t * n, flops=flops)
    # forward: q, k, v in, o out; backward: do in, dq, dk, dv out
    return dict(bytes=state * (2 if case["dtype"] == F32 else 1) + 2 * qk + 4 * val + 2 * gates + t * n,
                flops=3 * flops)


# ---------------------------------------------------------------- the definition in 64 bits
def exact(case, seed):
    st = prepare(case, seed)
    with torch.no_grad():
        if case["kind"].startswith("norm"):
            return _exact_norm(st)
        return _exact_delta(case, st)


def _exact_norm(st):
    rows, width = st["x"].shape
    wp, wq, r = (st[n].double() for n in ("w_post", "w_pre", "residual_scale"))
    train = "ds" in st
    per_channel = st["gate"].dim() == 1
    parts, sums = [], {}
    for at in range(0, rows, 1 << 14):
        cut = slice(at, min(rows, at + (1 << 14)))
        x, y = st["x"][cut].double(), st["y"][cut].double()
        gate = (st["gate"] if per_channel else st["gate"][cut]).double()
        ry = 1.0 / torch.sqrt((y * y).sum(1, keepdim=True) / width + st["eps"])
        s = r * x + gate * (y * ry * wp)
        rs = 1.0 / torch.sqrt((s * s).sum(1, keepdim=True) / width + st["eps"])
        part = dict(s=s, h=s * rs * wq)
        if train:
            dh = st["dh"][cut].double()
            z = dh * wq
            total = st["ds"][cut].double() + rs * z - s * rs ** 3 * ((z * s).sum(1, keepdim=True) / width)
            dn = total * gate * wp
            part["d_x"] = r * total
            part["d_y"] = ry * dn - y * ry ** 3 * ((dn * y).sum(1, keepdim=True) / width)
            dg = total * (y * ry * wp)
            per = dict(d_w_pre=dh * s * rs, d_w_post=total * gate * (y * ry), d_residual_scale=total * x)
            if per_channel:
                per["d_gate"] = dg
            else:
                part["d_gate"] = dg if st["gate"].shape[1] == width else dg.sum(1, keepdim=True)
            for name, value in per.items():
                sums[name] = sums.get(name, 0.0) + value.sum(0)
        parts.append(part)
    out = {name: torch.cat([p[name] for p in parts]) for name in parts[0]}
    return dict(out, **sums)


def _exact_delta(case, st):
    """Tick by tick, forward and in reverse, for some environments at a time."""
    kind, h, kd, vd = case["kind"], case["heads"], case["k"], case["v"]
    n, t, shared = case["envs"], case["ticks"], case["heads"] // case["qk_heads"]
    # a tick is about ten launches forward and thirty in reverse; the states of all ticks are kept for the reverse
    cells = h * kd * vd
    group = max(1, min(n, (1 << 28 if kind != "train" else (1 << 31) // (t + 8)) // cells))
    launches = -(-n // group) * t * (10 if kind != "train" else 40)
    if launches > 1200000:
        return None
    scale = kd ** -0.5
    found = {}

    def put(name, value):
        found.setdefault(name, []).append(value)

    for at in range(0, n, group):
        e = slice(at, min(n, at + group))
        step = kind == "step"
        q, k, v, g, b, first = ((st[x][None, e] if step else st[x][:, e]) for x in ("q", "k", "v", "g", "beta", "reset"))
        q, k = (x.double().repeat_interleave(shared, 2) for x in (q, k))
        v, b = v.double(), b.double()
        decay = torch.exp(g.double()) * (first == 0).double()[..., None]
        s = st["state"][e].double()
        o = torch.empty_like(v)
        states, writes = [], []
        for j in range(t):
            if kind == "train":
                states.append(s)
            sd = decay[j][..., None, None] * s
            e1 = v[j] - (k[j][..., None, :] @ sd)[..., 0, :]
            s = sd + k[j][..., None] * (b[j][..., None] * e1)[..., None, :]
            o[j] = scale * (q[j][..., None, :] @ s)[..., 0, :]
            if kind == "train":
                writes.append(e1)
        put("o", o[0] if step else o)
        if step or (kind == "scan" and st["final"]):
            put("state", s)
        if kind != "train":
            continue
        do = st["do"][:, e].double()
        dq, dk, dv = torch.empty_like(q), torch.empty_like(k), torch.empty_like(v)
        dg, db = torch.empty_like(decay), torch.empty_like(b)
        grad, after = torch.zeros_like(s), s
        for j in range(t - 1, -1, -1):
            sd = decay[j][..., None, None] * states[j]
            grad = grad + scale * q[j][..., None] * do[j][..., None, :]
            dq[j] = scale * (after @ do[j][..., None])[..., 0]
            u = b[j][..., None] * writes[j]
            du = (k[j][..., None, :] @ grad)[..., 0, :]
            dv[j] = b[j][..., None] * du
            db[j] = (du * writes[j]).sum(-1)
            dk[j] = (grad @ u[..., None])[..., 0] - (sd @ dv[j][..., None])[..., 0]
            grad = grad - k[j][..., None] * dv[j][..., None, :]
            dg[j] = (grad * sd).sum((-1, -2))
            grad = decay[j][..., None, None] * grad
            after = states[j]
        for name, value in (("d_q", dq), ("d_k", dk)):
            put(name, value.unflatten(2, (-1, shared)).sum(3))
        for name, value in (("d_v", dv), ("d_g", dg), ("d_beta", db)):
            put(name, value)
        if st["state"].requires_grad:
            put("d_state", grad)
    dims = dict(o=0 if kind == "step" else 1, state=0, d_state=0)
    return {name: torch.cat(parts, dims.get(name, 1)) for name, parts in found.items()}
