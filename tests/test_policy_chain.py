"""The operators of a recurrent policy as they are used together: observations through a linear layer, a memory and a
gated block with its norms, to logits and the clipped loss; and the same policy tick by tick.

Against the same network in float64, by torch's own automatic gradients.  Tolerances, set before the first run: fp32
operators are off by 1e-6 to 4e-6 of their result's norm each (their own tests), a dozen of them one after the other,
with norms and a softmax between that pass errors on about as they are: 1e-4 of a gradient's norm."""
import math

import pytest
import torch  # before the library: one HIP runtime in the process

gpu = pytest.mark.gpu
T, N, OBS, WIDTH, HEADS, DIM, HIDDEN, COMMANDS, LEVELS = 12, 37, 181, 64, 2, 16, 200, 4, 33


def weights(dtype, device):
    gen = torch.Generator().manual_seed(2)

    def randn(*shape, scale=1.0):
        return (scale * torch.randn(*shape, generator=gen)).to(dtype).to(device)

    w = dict(enc=randn(WIDTH, OBS, scale=OBS ** -0.5), b_enc=randn(WIDTH, scale=0.1), qkv=randn(3 * HEADS * DIM, WIDTH, scale=WIDTH ** -0.5),
             gates=randn(2 * HEADS, WIDTH, scale=WIDTH ** -0.5), out=randn(WIDTH, HEADS * DIM, scale=0.2), gate=randn(HIDDEN, WIDTH, scale=WIDTH ** -0.5),
             up=randn(HIDDEN, WIDTH, scale=WIDTH ** -0.5), b_gate=randn(HIDDEN, scale=0.1), b_up=randn(HIDDEN, scale=0.1),
             down=randn(WIDTH, HIDDEN, scale=HIDDEN ** -0.5), b_down=randn(WIDTH, scale=0.1), head=randn(COMMANDS * LEVELS, WIDTH, scale=0.3))
    for n in ("post", "pre"):
        w[n] = (1 + 0.1 * torch.randn(WIDTH, generator=gen)).to(device)
    return w


class Own:
    """The framework's operators."""

    def __init__(self):
        from mdnav import policy, sequence
        self.linear, self.gated, self.loss = policy.linear, policy.gated_feed_forward, policy.clipped_loss
        self.rule, self.tick, self.norm = sequence.delta_rule, sequence.delta_rule_step, sequence.block_norm


class Plain:
    """The same from elementary operations, in the type of what they are given."""

    @staticmethod
    def linear(x, w, b=None, activation=None, residual=None):
        y = x @ w.t() + (0 if b is None else b)
        y = torch.tanh(y) if activation == "tanh" else y
        return y if residual is None else residual + y

    @staticmethod
    def gated(x, wg, wu, bg, bu, activation):
        z = x @ wg.t() + bg
        return z / (1 + torch.exp(-z)) * (x @ wu.t() + bu)

    @staticmethod
    def norm(x, y, w_post, w_pre):
        n = y / torch.sqrt(y.square().mean(-1, keepdim=True) + 1e-6)
        s = x + n * w_post
        return s, s / torch.sqrt(s.square().mean(-1, keepdim=True) + 1e-6) * w_pre

    @staticmethod
    def rule(q, k, v, g, beta, reset):
        s, out = torch.zeros(N, HEADS, DIM, DIM, dtype=q.dtype, device=q.device), []
        for t in range(q.shape[0]):
            s = s * (torch.exp(g[t]) * ~reset[t][:, None])[..., None, None]
            u = beta[t][..., None] * (v[t] - (s * k[t][..., None]).sum(-2))
            s = s + k[t][..., None] * u[..., None, :]
            out.append((s * q[t][..., None]).sum(-2) * DIM ** -0.5)
        return torch.stack(out), None

    @staticmethod
    def loss(logits, actions, old, adv, ref_log_prob, mask, clip, kl_coef, entropy_coef):
        lp = torch.log_softmax(logits, -1)
        l = lp.gather(-1, actions[..., None])[..., 0].sum(-1)
        r, far = torch.exp(l - old), ref_log_prob - l
        each = -torch.minimum(r * adv, r.clamp(1 - clip, 1 + clip) * adv) + kl_coef * (torch.exp(far) - far - 1)
        return (each + entropy_coef * (torch.exp(lp) * lp).sum((-1, -2)))[mask].mean(), None


def logits(f, w, obs, reset, state=None):
    """[T][N][OBS] to logits, or one tick [N][OBS] with `state` advanced."""
    x = f.linear(obs, w["enc"], w["b_enc"], activation="tanh")
    q, k, v = f.linear(x, w["qkv"]).unflatten(-1, (3, HEADS, DIM)).unbind(-3)
    g, beta = f.linear(x, w["gates"]).unflatten(-1, (2, HEADS)).unbind(-2)
    q, k = (t / torch.sqrt(t.square().sum(-1, keepdim=True) + 1e-6) for t in (q, k))
    rows = (q, k, v, -torch.nn.functional.softplus(g - 2.0), torch.sigmoid(beta))
    o = f.rule(*rows, reset=reset)[0] if state is None else f.tick(*rows, state, reset=reset)
    s, h = f.norm(x, f.linear(o.flatten(-2), w["out"]), w["post"], w["pre"])
    a = f.gated(h, w["gate"], w["up"], w["b_gate"], w["b_up"], activation="silu")
    y = f.linear(a, w["down"], w["b_down"], residual=s)
    return f.linear(y, w["head"]).unflatten(-1, (COMMANDS, LEVELS))


def data(device):
    gen = torch.Generator().manual_seed(3)
    l0 = -COMMANDS * math.log(LEVELS)
    return dict(obs=torch.randn(T, N, OBS, generator=gen).to(device), reset=(torch.rand(T, N, generator=gen) < 0.1).to(device),
                actions=torch.randint(LEVELS, (T, N, COMMANDS), generator=gen).to(device),
                old=(l0 + 0.5 * torch.randn(T, N, generator=gen)).to(device), adv=torch.randn(T, N, generator=gen).to(device),
                ref=(l0 + 0.5 * torch.randn(T, N, generator=gen)).to(device), mask=(torch.rand(T, N, generator=gen) > 0.1).to(device))


def train(f, w, d, dtype):
    leaves = {n: t.detach().to(dtype).requires_grad_() for n, t in w.items()}
    z = logits(f, leaves, d["obs"].to(dtype), d["reset"])
    kind = torch.float64 if dtype == torch.float64 else torch.float32
    old, adv, ref = (d[n].to(kind) for n in ("old", "adv", "ref"))
    # ratios near 1, as after some updates
    l = torch.log_softmax(z.detach().double(), -1).gather(-1, d["actions"][..., None])[..., 0].sum(-1)
    shift = (l + COMMANDS * math.log(LEVELS)).to(kind)
    loss, _ = f.loss(z, d["actions"], old + shift, adv, ref_log_prob=ref + shift, mask=d["mask"], clip=0.2, kl_coef=0.05, entropy_coef=0.01)
    return z, loss, torch.autograd.grad(loss, list(leaves.values()))


@gpu
def test_a_training_step_and_its_ticks():
    d, w = data("cuda"), weights(torch.float32, "cuda")
    z, loss, grads = train(Own(), w, d, torch.float32)
    want_z, want_loss, want = train(Plain(), w, d, torch.float64)
    assert (z.double() - want_z).norm() < 1e-5 * want_z.norm() and abs(loss.item() - want_loss.item()) < 1e-5
    for n, a, b in zip(w, grads, want):
        off = ((a.double() - b).norm() / b.norm()).item()
        print("  d_%s: %.2e" % (n, off), flush=True)
        assert off < 1e-4, n
    # tick by tick, and what acting stores
    from mdnav import policy
    state = torch.zeros(N, HEADS, DIM, DIM, device="cuda")
    with torch.no_grad():
        for t in range(T):
            now = logits(Own(), w, d["obs"][t], d["reset"][t], state)
            assert (now - z[t]).norm() < 1e-5 * z[t].norm()
            l, h = policy.log_prob(now, d["actions"][t])
            lp = torch.log_softmax(want_z[t], -1)
            assert (l - lp.gather(-1, d["actions"][t][..., None])[..., 0].sum(-1)).abs().max() < 1e-4
            assert (h + (lp * torch.exp(lp)).sum((-1, -2))).abs().max() < 1e-4


@gpu
def test_in_bfloat16():
    """Rows and weights in bfloat16: each of a dozen operators rounds to 2^-8, which random signs and norms leave as
    2^-8 sqrt(12) of the logits' norm; gradients go through as many again."""
    d, w = data("cuda"), weights(torch.bfloat16, "cuda")
    own, plain = Own(), Plain()

    def mixed(w):  # the norms' weights stay in 32 bits
        return {n: t.float() if n in ("post", "pre") else t for n, t in w.items()}

    leaves = {n: t.detach().requires_grad_() for n, t in mixed(w).items()}
    z = logits(own, leaves, d["obs"].bfloat16(), d["reset"])
    loss, _ = own.loss(z, d["actions"], d["old"], d["adv"], ref_log_prob=d["ref"], mask=d["mask"], clip=10.0, kl_coef=0.0, entropy_coef=0.01)
    grads = torch.autograd.grad(loss, list(leaves.values()))
    exact = {n: t.double().detach().requires_grad_() for n, t in w.items()}
    want_z = logits(plain, exact, d["obs"].bfloat16().double(), d["reset"])
    # (a clip of 10 and no reference: the loss does not jump)
    want_loss, _ = plain.loss(want_z, d["actions"], d["old"].double(), d["adv"].double(), ref_log_prob=d["ref"].double(), mask=d["mask"],
                              clip=10.0, kl_coef=0.0, entropy_coef=0.01)
    assert (z.double() - want_z).norm() < 2.0 ** -8 * 12 ** 0.5 * want_z.norm()
    # A step's slope is A r with r = exp(l - old): l is off by the logits' own error, 2^-8 sqrt(12) of their size, from
    # each of the commands, and r by as much of itself.
    size = want_z.detach().square().mean().sqrt().item()
    room = 2.0 ** -8 * (2 * 24 ** 0.5 + 12 ** 0.5 * size * COMMANDS ** 0.5)
    for n, a, b in zip(w, grads, torch.autograd.grad(want_loss, list(exact.values()))):
        off = ((a.double() - b).norm() / b.norm()).item()
        print("  d_%s: %.2e" % (n, off), flush=True)
        assert off < room, n


@gpu
def test_a_captured_training_step():
    d, w = data("cuda"), weights(torch.float32, "cuda")

    def step():
        z, loss, grads = train(Own(), w, d, torch.float32)
        return [z.detach(), loss.detach(), *grads]

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    gen = torch.Generator(device="cuda").manual_seed(5)
    for _ in range(4):
        d["obs"].copy_(torch.randn(T, N, OBS, generator=gen, device="cuda"))
        w["gate"].mul_(0.9)
        want = [t.clone() for t in step()]
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)
