"""The sequence operators in a captured HIP graph: replays give what eager calls give."""
import pytest
import torch


@pytest.mark.gpu
@pytest.mark.parametrize("ticks,envs,width", [(70, 9, 64), (600, 2, 128)], ids=["chunks", "segments"])
def test_a_captured_step_and_rollout(ticks, envs, width):
    from mdnav import sequence
    gen = torch.Generator(device="cuda").manual_seed(5)

    def normal(*shape):
        return torch.randn(*shape, generator=gen, device="cuda")

    def fill():
        for t in (q, k, v, x, y):
            t.copy_(normal(*t.shape) * width ** -0.5)
        g.copy_(-normal(*g.shape).abs() * 0.1)
        beta.copy_(torch.sigmoid(normal(*beta.shape)))
        state.copy_(normal(*state.shape))
        moving.copy_(state)

    q, k, v = (torch.empty(ticks, envs, 1, width, device="cuda", dtype=torch.bfloat16) for _ in range(3))
    g, beta = (torch.empty(ticks, envs, 1, device="cuda") for _ in range(2))
    x, y = (torch.empty(ticks, envs, width, device="cuda") for _ in range(2))
    weight = torch.rand(width, generator=gen, device="cuda")
    state, moving = (torch.empty(envs, 1, width, width, device="cuda") for _ in range(2))

    def calls():
        o, last = sequence.delta_rule(q, k, v, g, beta, state=state, final_state=True)
        one = sequence.delta_rule_step(q[0], k[0], v[0], g[0], beta[0], moving)
        s, h = sequence.block_norm(x, y, weight, weight)
        return [o, last, one, s, h, moving]

    fill()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        calls()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = calls()
    for _ in range(4):
        fill()
        want = [t.clone() for t in calls()]
        moving.copy_(state)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(captured, want):
            assert torch.equal(a, b)
