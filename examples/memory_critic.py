"""A critic with a learned memory, trained on the rollouts of a Sim.

A fleet's actor observations show one moment of a flight.  This critic keeps a
matrix of what an environment has seen (the gated delta rule, one state of
64 x 64 per environment and head) and learns to predict the rollout's returns
from actor observations alone:

* training takes whole rollouts: ``delta_rule`` over [ticks][envs] rows, with
  the episodes that end inside, its gradients and those of ``block_norm``;
* acting takes one tick: ``delta_rule_step`` advances the fleet's states in
  place, which are then those that the rollout's last tick left.

    python examples/memory_critic.py --envs 1024 --horizon 64 --rollouts 8
"""
import argparse
import os
import sys

import torch
import torch.nn.functional as F

sys.path.insert(0, os.path.join(os.path.dirname(os.path.abspath(__file__)), "..", "metal-drone-nav_amd"))
from mdnav import PPOTrainer, Sim, abi, sequence  # noqa: E402


class MemoryCritic(torch.nn.Module):
    def __init__(self, obs, width=128, heads=2, head_dim=64, dtype=torch.float32):
        super().__init__()
        self.heads, self.head_dim, self.dtype = heads, head_dim, dtype
        self.stream = torch.nn.Linear(obs, width, dtype=dtype)      # what the residual stream starts with
        self.embed = torch.nn.Linear(obs, width, dtype=dtype)       # the first block
        self.qkv = torch.nn.Linear(width, 3 * heads * head_dim, bias=False, dtype=dtype)
        self.gates = torch.nn.Linear(width, 2 * heads, dtype=dtype)
        self.out = torch.nn.Linear(heads * head_dim, width, bias=False, dtype=dtype)
        self.value = torch.nn.Linear(width, 1, dtype=dtype)
        torch.nn.init.zeros_(self.value.weight)
        torch.nn.init.zeros_(self.value.bias)
        for name in ("w_post1", "w_pre1", "w_post2", "w_pre2", "scale"):
            setattr(self, name, torch.nn.Parameter(torch.ones(width)))
        self.block_gate = torch.nn.Parameter(torch.full((width,), 0.5))

    def rows(self, obs):
        """The stream and the memory's inputs, of any rows."""
        x, h = sequence.block_norm(self.stream(obs), torch.tanh(self.embed(obs)), self.w_post1, self.w_pre1)
        q, k, v = self.qkv(h).unflatten(-1, (3, self.heads, self.head_dim)).unbind(-3)
        g, beta = self.gates(h).float().unflatten(-1, (2, self.heads)).unbind(-2)
        # a decay of about 0.98 a tick to begin with
        return x, F.normalize(q, dim=-1), F.normalize(k, dim=-1), v, -F.softplus(g - 4.0), torch.sigmoid(beta)

    def values(self, x, o):
        y = self.out(o.flatten(-2))
        _, h = sequence.block_norm(x, y, self.w_post2, self.w_pre2, gate=self.block_gate, residual_scale=self.scale)
        return self.value(h).squeeze(-1).float()

    def forward(self, obs, reset, state):
        """Whole rollouts: obs [ticks][envs][..], reset [ticks][envs], state before the first tick."""
        x, *memory = self.rows(obs)
        o, state = sequence.delta_rule(*memory, state=state, reset=reset, final_state=True)
        return self.values(x, o), state

    @torch.no_grad()
    def step(self, obs, reset, state):
        """One tick: obs [envs][..], reset [envs]; ``state`` is advanced in place."""
        x, *memory = self.rows(obs)
        return self.values(x, sequence.delta_rule_step(*memory, state, reset=reset))

    def new_state(self, envs, device):
        return torch.zeros(envs, self.heads, self.head_dim, self.head_dim, device=device)


def rollout_rows(sim, ended, device):
    """The last rollout's observations, returns and first ticks of episodes.
    ``ended``: the envs whose episode the rollout before this one ended."""
    t, n = sim.horizon, sim.n
    obs = torch.from_numpy(sim.get("obs").reshape(t, n, -1)).to(device)
    returns = torch.from_numpy(sim.get("returns").reshape(t, n)).to(device)
    done = torch.from_numpy(sim.get("terminated") | sim.get("truncated")).reshape(t, n).to(device) != 0
    return obs, returns, torch.cat([ended[None], done[:-1]]), done[-1]


def train(envs=1024, horizon=64, rollouts=8, epochs=8, lr=3e-4, dtype=torch.float32, seed=1, log=print):
    """Returns the critic, the losses of every rollout's first and last epoch,
    and the largest difference between the last rollout's values made at once
    and tick by tick."""
    device = torch.device("cuda")
    torch.manual_seed(seed)
    sim = Sim(abi.default_config(n=envs, family=1, speed=1.0, distance=3.0, seed=seed), horizon=horizon)
    ppo = PPOTrainer(sim, epochs=1, minibatch=envs * horizon // 4)
    critic = MemoryCritic(sim.actor_obs, dtype=dtype).to(device)
    optimizer = torch.optim.Adam(critic.parameters(), lr=lr)
    state, ended, losses = critic.new_state(envs, device), torch.ones(envs, dtype=torch.bool, device=device), []
    for r in range(rollouts):
        sim.collect()
        ppo.gae()
        sim.sync()
        obs, returns, reset, next_ended = rollout_rows(sim, ended, device)
        obs = obs.to(dtype)
        for epoch in range(epochs):
            values, last = critic(obs, reset, state)
            loss = F.mse_loss(values, returns)
            optimizer.zero_grad(set_to_none=True)
            loss.backward()
            torch.nn.utils.clip_grad_norm_(critic.parameters(), 1.0)
            optimizer.step()
            if epoch == 0:
                first = loss.item()
        losses.append((first, loss.item()))
        log("rollout %d: loss %.4f -> %.4f, returns' variance %.4f" % (r, *losses[-1], returns.var().item()), flush=True)
        with torch.no_grad():
            values, last = critic(obs, reset, state)
        if r + 1 == rollouts:
            ticks = torch.stack([critic.step(obs[t], reset[t], state) for t in range(horizon)])
            differ = max((ticks - values).abs().max().item(), (state - last).abs().max().item())
        state, ended = last, next_ended
    ppo.close()
    sim.close()
    return critic, losses, differ


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description="a critic with a learned memory on rollouts of a fleet")
    parser.add_argument("--envs", type=int, default=1024)
    parser.add_argument("--horizon", type=int, default=64)
    parser.add_argument("--rollouts", type=int, default=8)
    parser.add_argument("--epochs", type=int, default=8)
    parser.add_argument("--bf16", action="store_true", help="rows and weights in bfloat16; states stay in 32 bits")
    args = parser.parse_args()
    _, _, differ = train(args.envs, args.horizon, args.rollouts, args.epochs,
                         dtype=torch.bfloat16 if args.bf16 else torch.float32)
    print("tick by tick: values and states within %.2g of the rollout's" % differ)
