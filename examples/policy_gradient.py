"""A policy trained on sliding-tile environments, on the device end to end.

Each step: the environments' states become tokens (their true atoms), the applicable actions those of ``rl.expand``;
``learn.embedding`` looks both up, a small network gives a logit for each action, ``learn.logprobs`` the log-probability
and the entropy over each state's own actions; an action is drawn and the environments step. After a few steps a
REINFORCE loss on the discounted rewards to come, with an entropy bonus, goes back through both into ``learn.AdamW``
(moments in 8 bits).

    python examples/policy_gradient.py --envs 2048 --updates 60
"""

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))

import torch

from mymyr_b200 import learn, rl, tasks
from mymyr_b200.task import Task


def true_atoms(states: torch.Tensor, slots: int, most: int) -> torch.Tensor:
    """The true atoms of packed states [N, W], ascending, as tokens [N, most]; -1 past a state's last."""
    word = torch.arange(slots, device=states.device)
    bits = states[:, word >> 6] >> (word & 63) & 1
    order = torch.argsort(bits, dim=1, descending=True, stable=True)[:, :most]
    return torch.where(bits.gather(1, order) > 0, order, -1)


class Policy:
    """Embedded atoms and actions, two layers, a logit for each action."""

    def __init__(self, task: Task, width: int, device, dtype=torch.float32):
        g = torch.Generator(device=device).manual_seed(0)

        def normal(*shape, scale):
            return (torch.randn(*shape, generator=g, device=device) * scale).to(dtype).requires_grad_(True)

        self.task = task
        self.atoms = normal(task.fluent_slots, width, scale=0.1)
        # an action is its schema's token and one token for each (position, object)
        self.labels = normal(task.num_schemas + task.label_width * task.num_objects, width, scale=0.1)
        self.hidden = normal(2 * width, width, scale=(2 * width) ** -0.5)
        self.out = normal(width, 1, scale=width ** -0.5)

    def parameters(self):
        return [self.atoms, self.labels, self.hidden, self.out]

    def logits(self, states: torch.Tensor, e: rl.Expansion, most: int) -> torch.Tensor:
        """[M]: a logit for each successor of the expansion."""
        t = self.task
        atoms = learn.embedding(true_atoms(states, t.fluent_slots, most), self.atoms).sum(1)
        place = torch.arange(e.binding.shape[1], device=states.device) * t.num_objects + t.num_schemas
        label = torch.where(e.binding >= 0, e.binding + place, -1)
        label = torch.cat((e.schema[:, None].long(), label), 1)
        action = learn.embedding(label, self.labels).sum(1)
        x = torch.cat((atoms[e.parent.long()], action), 1)
        return ((x @ self.hidden).tanh() @ self.out).squeeze(1)


def draw(logits: torch.Tensor, offsets: torch.Tensor, generator) -> torch.Tensor:
    """An action of each state in proportion to its probability: the largest of its logits plus Gumbel noise. -1 where
    there is none."""
    u = torch.rand(logits.shape, generator=generator, device=logits.device).clamp_(1e-9, 1 - 1e-7)
    return learn.logprobs(logits.detach() - (-u.log()).log(), offsets=offsets, top=1).top_tokens[:, 0]


def train(envs: int = 2048, updates: int = 60, horizon: int = 8, width: int = 64, side: int = 3, scramble: int = 6,
          seed: int = 0, log=print) -> list[float]:
    """Returns the mean reward of a step in each update's rollout."""
    task = Task.from_text(tasks.sliding_tile(side, side, scramble, seed))
    env = rl.BatchedEnv(task, envs, seed=seed, max_steps=32)
    env.reset()
    device = env.states.device
    most = side * side + 1  # each tile's place and the blank's
    policy = Policy(task, width, device)
    opt = learn.AdamW(policy.parameters(), lr=3e-3, weight_decay=0.0, bits=8)
    generator = torch.Generator(device=device).manual_seed(seed)
    means = []
    for update in range(updates):
        steps = []
        for _ in range(horizon):
            e = rl.expand(task, env.states, hashes=False)
            logits = policy.logits(env.states, e, most)
            action = draw(logits, e.offsets, generator)
            got = learn.logprobs(logits, action, offsets=e.offsets)
            env.step(action.clamp(min=0))
            over = (env.terminated | env.truncated).bool()
            steps.append((got.logprob, got.entropy, env.reward.clone(), over.clone()))
        loss, to_come = 0.0, torch.zeros(envs, device=device)
        for logprob, entropy, reward, over in reversed(steps):
            to_come = reward + 0.9 * torch.where(over, 0.0, to_come)
            loss = loss - (logprob * (to_come - to_come.mean())).mean() - 0.01 * entropy.mean()
        opt.zero_grad()
        loss.backward()
        opt.step()
        means.append(float(torch.stack([r for _, _, r, _ in steps]).mean()))
        if update % 10 == 0 or update == updates - 1:
            entropy = float(torch.stack([h for _, h, _, _ in steps]).detach().mean())
            log(f"update {update}: mean reward of a step {means[-1]:.4f}, entropy {entropy:.3f}")
    env.check_errors()
    return means


if __name__ == "__main__":
    ap = argparse.ArgumentParser(description=__doc__.splitlines()[0])
    ap.add_argument("--envs", type=int, default=2048)
    ap.add_argument("--updates", type=int, default=60)
    ap.add_argument("--horizon", type=int, default=8)
    ap.add_argument("--width", type=int, default=64)
    ap.add_argument("--side", type=int, default=3)
    ap.add_argument("--scramble", type=int, default=6)
    a = ap.parse_args()
    train(a.envs, a.updates, a.horizon, a.width, a.side, a.scramble)
