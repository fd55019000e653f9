"""Gradients that reach a backward pass lazily negated, as those of a complex number's imaginary part do behind a
conjugate: torch keeps the values and a flag, and what reads the memory has to have the flag taken off first."""
import ctypes

import pytest
import torch  # before the library: one HIP runtime in the process

gpu = pytest.mark.gpu


def negated(t):
    """`t` as memory that holds -t and a flag."""
    out = torch._neg_view(-t)
    assert out.is_neg() and torch.equal(out, t)
    return out


def floats(address, count):
    return list((ctypes.c_float * count).from_address(address))


class _Library:
    """Stands in for the library on the CPU: notes the gradients that the backward entries are given."""

    def __init__(self):
        self.seen = []

    def __call__(self):
        return self

    def __getattr__(self, name):
        return lambda *args: 0

    def mdn_op_choices_loss_sizes(self, choices, keep, workspace):
        keep._obj.value = 16
        return 0

    def mdn_op_dense_backward(self, dense, grad, *_):
        d_y = grad._obj.d_y
        self.seen.append([floats(d_y.data + 4 * d_y.row * i, dense._obj.out) for i in range(dense._obj.rows)])
        return 0

    def mdn_op_choices_loss_backward(self, choices, loss, keep, size, d_loss, *_):
        self.seen.append(floats(d_loss, 1))
        return 0


@pytest.fixture
def library(monkeypatch):
    from mdnav import policy
    monkeypatch.setattr(policy, "_device", lambda names, tensors: torch.device("cpu"))
    monkeypatch.setattr(policy, "_on", lambda device, f, *args: f(*args))
    monkeypatch.setattr(policy, "_stream", lambda device: None)
    library = _Library()
    monkeypatch.setattr(policy, "_library", library)
    return library


@pytest.mark.parametrize("width", [1, 6])
def test_a_layer_sees_the_values(library, width):
    from mdnav import policy
    x, w, d_y = torch.randn(4, 3, requires_grad=True), torch.randn(width, 3, requires_grad=True), torch.randn(4, width)
    for f in (lambda: policy.linear(x, w), lambda: policy.gated_feed_forward(x, w, w)):
        torch.autograd.grad(f(), x, negated(d_y))
        # as it comes about: the imaginary part's gradient, two floats apart
        y = f()
        y = torch.complex(torch.zeros_like(y), torch.zeros_like(y) + (y - y.detach()))
        torch.autograd.grad(y.conj(), x, torch.complex(torch.zeros_like(d_y), -d_y))
    assert library.seen == 4 * [d_y.tolist()]


def test_a_loss_sees_the_value(library):
    from mdnav import policy
    logits = torch.randn(5, 2, 3, requires_grad=True)
    loss, _ = policy.clipped_loss(logits, torch.zeros(5, 2, dtype=torch.int64), torch.zeros(5), torch.zeros(5))
    torch.autograd.grad(loss, logits, negated(torch.tensor(3.0)))
    assert library.seen == [[3.0]]


@gpu
def test_policy_gradients():
    """The bits of gradients without the flag."""
    from mdnav import policy
    gen = torch.Generator().manual_seed(1)

    def randn(*shape):
        return torch.randn(*shape, generator=gen).cuda()

    for rows, width in ((300, 1), (300, 24)):
        x, w, u, d_y = randn(rows, 16).requires_grad_(), randn(width, 16).requires_grad_(), randn(width, 16), randn(rows, width)
        for f in (lambda: policy.linear(x, w), lambda: policy.linear(x, w, activation="tanh"), lambda: policy.gated_feed_forward(x, w, u)):
            for a, b in zip(torch.autograd.grad(f(), [x, w], negated(d_y)), torch.autograd.grad(f(), [x, w], d_y)):
                assert torch.equal(a, b)
    logits = randn(40, 2, 7).requires_grad_()
    data = torch.zeros(40, 2, dtype=torch.int64, device="cuda"), randn(40) - 4.0, randn(40)
    grads = []
    for d_loss in (negated(torch.tensor(3.0, device="cuda")), torch.tensor(3.0, device="cuda")):
        grads.append(torch.autograd.grad(policy.clipped_loss(logits, *data)[0], logits, d_loss)[0])
    assert grads[0].any() and torch.equal(*grads)


class _Sequence(_Library):
    def mdn_op_delta_rule_sizes(self, rule, sizes):
        sizes._obj.keep = 16
        return 0

    def mdn_op_delta_rule_backward(self, rule, grad, *_):
        r, d_o = rule._obj, grad._obj.d_o
        self.seen.append([[floats(d_o.data + 4 * (t * d_o.tick + n * d_o.env), r.v_dim) for n in range(r.envs)] for t in range(r.ticks)])
        self.seen.append(floats(grad._obj.d_state_out, r.envs * r.k_dim * r.v_dim))
        return 0

    def mdn_op_block_norm_backward(self, norm, grad, *_):
        for m in (grad._obj.d_s, grad._obj.d_h):
            self.seen.append([floats(m.data + 4 * m.inner * i, norm._obj.width) for i in range(norm._obj.rows)])
        return 0


@pytest.mark.parametrize("width", [1, 4])
def test_a_memory_and_norms_see_the_values(monkeypatch, width):
    from mdnav import sequence
    library = _Sequence()
    monkeypatch.setattr(sequence, "_device", lambda names, tensors: torch.device("cpu"))
    monkeypatch.setattr(sequence, "_on", lambda device, f, *args: f(*args))
    monkeypatch.setattr(sequence, "_stream", lambda device: None)
    monkeypatch.setattr(sequence, "_library", library)
    q, k, gate = torch.randn(3, 2, 1, 5), torch.randn(3, 2, 1, 5), torch.rand(3, 2, 1)
    v = torch.randn(3, 2, 1, width, requires_grad=True)
    d_o, d_last = torch.randn(3, 2, 1, width), torch.randn(2, 1, 5, width)
    out = sequence.delta_rule(q, k, v, -gate, gate, final_state=True)
    torch.autograd.grad(out, v, [negated(d_o), negated(d_last)])
    assert library.seen == [d_o[:, :, 0].tolist(), d_last.flatten().tolist()]
    library.seen.clear()
    x, w, d_s, d_h = torch.randn(6, width, requires_grad=True), torch.ones(width), torch.randn(6, width), torch.randn(6, width)
    torch.autograd.grad(sequence.block_norm(x, torch.randn(6, width), w, w), x, [negated(d_s), negated(d_h)])
    assert library.seen == [d_s.tolist(), d_h.tolist()]


@gpu
@pytest.mark.parametrize("width", [1, 16])
def test_sequence_gradients(width):
    """The bits of gradients without the flag."""
    from mdnav import sequence
    gen = torch.Generator().manual_seed(2)

    def randn(*shape):
        return torch.randn(*shape, generator=gen).cuda()

    q, k, gate = 0.3 * randn(40, 3, 1, 16), 0.3 * randn(40, 3, 1, 16), torch.sigmoid(randn(40, 3, 1))
    v, d_o, d_last = randn(40, 3, 1, width).requires_grad_(), randn(40, 3, 1, width), randn(3, 1, 16, width)
    grads = [torch.autograd.grad(sequence.delta_rule(q, k, v, -gate, gate, final_state=True), v, d)[0]
             for d in ([negated(d_o), negated(d_last)], [d_o, d_last])]
    assert grads[0].any() and torch.equal(*grads)
    x, y, w, d_s, d_h = randn(30, width).requires_grad_(), randn(30, width).requires_grad_(), randn(width), randn(30, width), randn(30, width)
    for a, b in zip(*[torch.autograd.grad(sequence.block_norm(x, y, w, w), [x, y], d) for d in ([negated(d_s), negated(d_h)], [d_s, d_h])]):
        assert torch.equal(a, b)
