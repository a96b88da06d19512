"""The example that trains a policy with the learner's operators over batched environments."""

import sys
from pathlib import Path

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

sys.path.insert(0, str(Path(__file__).resolve().parent.parent / "examples"))

import policy_gradient  # noqa: E402

from mymyr_b200 import learn, rl, tasks  # noqa: E402
from mymyr_b200.task import Task  # noqa: E402


def test_true_atoms_are_the_states_bits():
    task = Task.from_text(tasks.sliding_tile(3, 3, 12, 0))
    env = rl.BatchedEnv(task, 50, seed=0)
    env.reset()
    for _ in range(3):
        env.step()
    tokens = policy_gradient.true_atoms(env.states, task.fluent_slots, 12)
    words = env.states.cpu().numpy().view("uint64")
    for row, got in zip(words, tokens.tolist()):
        bits = [i for i in range(task.fluent_slots) if int(row[i // 64]) >> (i % 64) & 1]
        assert got == bits + [-1] * (12 - len(bits))


def test_actions_are_drawn_in_proportion():
    """60,000 rows of three logits: frequencies within five standard deviations of the probabilities."""
    n, p = 60000, torch.tensor([0.2, 0.5, 0.3], device="cuda")
    g = torch.Generator(device="cuda").manual_seed(1)
    offsets = torch.arange(0, 3 * n + 1, 3, device="cuda")
    got = policy_gradient.draw(p.log().repeat(n), offsets, g)
    freq = torch.bincount(got, minlength=3).double() / n
    assert ((freq - p).abs() < 5 * (p * (1 - p) / n).sqrt()).all()
    empty = policy_gradient.draw(torch.zeros(0, device="cuda"), torch.zeros(4, dtype=torch.int64, device="cuda"), g)
    assert empty.tolist() == [-1, -1, -1]


def test_the_policy_learns():
    """The reward of a step at the end is more than twice that of the first rollouts."""
    means = policy_gradient.train(envs=1024, updates=40, log=lambda *_: None)
    first, last = sum(means[:3]) / 3, sum(means[-3:]) / 3
    assert last > 2 * first, (first, last)
