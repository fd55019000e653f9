"""mdnav.sequence under torch's modes: what a program sets for all of its tensors, and derivatives that the
operators have none of."""
import pytest
import torch  # before the library: one HIP runtime in the process

gpu = pytest.mark.gpu


@pytest.fixture(params=[torch.bfloat16, torch.float16, torch.float64], ids=str)
def default_dtype(request):
    before = torch.get_default_dtype()
    torch.set_default_dtype(request.param)
    yield request.param
    torch.set_default_dtype(before)


class _NoLibrary:
    """Stands in for the library on the CPU: every call succeeds and does nothing."""

    def __getattr__(self, name):
        return lambda *args: 0


@pytest.fixture
def on_the_cpu(monkeypatch):
    from mdnav import sequence
    monkeypatch.setattr(sequence, "_device", lambda names, tensors: torch.device("cpu"))
    monkeypatch.setattr(sequence, "_library", _NoLibrary)
    monkeypatch.setattr(sequence, "_stream", lambda device: None)
    return sequence


def test_buffers_have_the_kernels_types(on_the_cpu, default_dtype):
    """What the kernels write as 32-bit floats is allocated as such, whatever torch's default type is."""
    f32 = torch.float32
    rows = torch.zeros(2, 3, 1, 4, dtype=torch.bfloat16)
    gates = torch.zeros(2, 3, 1, dtype=f32)
    call = on_the_cpu._Call(rows, rows, rows, gates, gates, torch.zeros(3, 1, 4, 4, dtype=f32), None, None)
    assert call.states().dtype == f32
    kept, sizes = call.forward(call.output(), call.states(), True)
    grads = call.backward(kept, sizes, rows, None, True)
    assert [g.dtype for g in grads] == 3 * [torch.bfloat16] + 3 * [f32]
    x, w = torch.zeros(3, 8, dtype=torch.bfloat16), torch.zeros(8, dtype=f32)
    call = on_the_cpu._NormCall(x, x, w, w, w, w, 1e-6)
    s, h, stats = call.forward(True)
    assert (s.dtype, h.dtype, stats.dtype) == (torch.bfloat16, torch.bfloat16, f32)
    d_x, d_y, *sums = call.backward(stats, x, x)
    assert [g.dtype for g in (d_x, d_y)] == 2 * [torch.bfloat16] and all(g.dtype == f32 for g in sums)


@gpu
def test_another_default_type_changes_nothing(default_dtype):
    """Results and gradients have the same types and bits as under torch's own default."""
    from mdnav import sequence
    gen = torch.Generator().manual_seed(2)

    def randn(*shape):
        return torch.randn(*shape, generator=gen, dtype=torch.float32).cuda()

    rule = [0.3 * randn(40, 3, 2, 16).bfloat16(), 0.3 * randn(40, 3, 2, 16).bfloat16(), randn(40, 3, 2, 24).bfloat16(),
            -randn(40, 3, 2).abs(), torch.sigmoid(randn(40, 3, 2)), randn(3, 2, 16, 24)]
    norm = [randn(50, 40), randn(50, 40), randn(40), randn(40)]
    runs = []
    for dtype in (torch.float32, default_dtype):
        torch.set_default_dtype(dtype)
        leaves = [t.detach().requires_grad_() for t in rule + norm]
        o, last = sequence.delta_rule(*leaves[:6], final_state=True)
        s, h = sequence.block_norm(*leaves[6:], gate=leaves[8], residual_scale=leaves[9])
        assert last.dtype == torch.float32
        outs = [o, last, s, h]
        runs.append(outs + list(torch.autograd.grad(outs, leaves, [torch.ones_like(t) for t in outs])))
    for a, b in zip(*runs):
        assert a.dtype == b.dtype and torch.equal(a, b)


def test_forward_mode_derivatives_are_refused():
    """A dual tensor has a tangent that no result would have: every operator raises for one in any argument,
    with and without gradients of other arguments, and takes plain tensors at the same level as ever."""
    import torch.autograd.forward_ad as forward_ad
    from mdnav import sequence
    rows, gates, state, weight = torch.zeros(2, 3, 1, 4), torch.zeros(2, 3, 1), torch.zeros(3, 1, 4, 4), torch.ones(4)
    calls = ((sequence.delta_rule, [rows, rows, rows, gates, gates, state]),
             (sequence.delta_rule_step, [rows[0], rows[0], rows[0], gates[0], gates[0], state]),
             (sequence.block_norm, [rows, rows, weight, weight, weight, weight]))
    for call, args in calls:
        for i in range(len(args)):
            for grad in (False, True):
                with forward_ad.dual_level():
                    some = [a.clone() for a in args]
                    some[i - 1].requires_grad_(grad and i > 0)
                    some[i] = forward_ad.make_dual(some[i], torch.ones_like(some[i]))
                    with pytest.raises(NotImplementedError, match="forward-mode"):
                        call(*some)
                    with torch.no_grad(), pytest.raises(NotImplementedError, match="forward-mode"):
                        call(*some)
        with forward_ad.dual_level(), pytest.raises(ValueError, match="GPU"):
            call(*args)


def test_numbers_that_want_gradients_are_refused():
    """``scale`` and ``eps`` are numbers; a learned one would silently get no gradient."""
    from mdnav import sequence
    rows, gates, state, weight = torch.zeros(2, 3, 1, 4), torch.zeros(2, 3, 1), torch.zeros(3, 1, 4, 4), torch.ones(4)
    learned = torch.tensor(0.5, requires_grad=True)
    calls = (lambda x: sequence.delta_rule(rows, rows, rows, gates, gates, scale=x),
             lambda x: sequence.delta_rule_step(rows[0], rows[0], rows[0], gates[0], gates[0], state, scale=x),
             lambda x: sequence.block_norm(rows, rows, weight, weight, eps=x))
    for call in calls:
        with pytest.raises(TypeError, match="is a number"):
            call(learned)
        with torch.no_grad(), pytest.raises(ValueError, match="GPU"):
            call(learned)
        with pytest.raises(ValueError, match="GPU"):
            call(learned.detach())
