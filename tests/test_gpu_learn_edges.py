"""The learner's operators where they went wrong once, or could: buffers of the caller's own, empty calls, numbers at the
ends of their range, steps that differ from parameter to parameter, arrays past 2^32 elements.

Tolerances come from the roundings a value goes through, EPS = 2^-24 each (32-bit arithmetic)."""

import ctypes as C
import math

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from mymyr_b200 import _lib, learn  # noqa: E402
from mymyr_b200.task import default_context  # noqa: E402

INF = float("inf")
EPS = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def randn(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale


# ------------------------------------------------------------------------------------------------ AdamW

def shifted(t, by):
    """The same numbers, `by` elements into a buffer of their own."""
    buffer = torch.zeros(t.numel() + by, dtype=torch.uint8 if t.element_size() == 1 else t.dtype, device=t.device)
    buffer = buffer.view(t.dtype)
    part = buffer[by:]
    part.view(torch.uint8).copy_(t.view(torch.uint8))
    return part


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_refuses_moments_off_a_vector_boundary(bits):
    """Host check: nothing is launched, and nothing changes. At a boundary of eight elements the same call is taken."""
    names = ("exp_avg", "exp_avg_sq", "master")
    p = randn(600, seed=1).bfloat16()
    before = p.clone()
    g = randn(600, seed=2).bfloat16()
    state = learn.adamw_state([p], bits=bits, master=True)
    for name in names:
        for by in (1, 4):
            with pytest.raises(ValueError, match="boundary"):
                learn.adamw_step([p], [g], step=1, **(state | {name: shifted(state[name], by)}))
    assert torch.equal(p, before)
    moved = {k: shifted(t, 8) if k in names else t for k, t in state.items()}
    learn.adamw_step([p], [g], step=1, **moved)
    other = learn.adamw_state([before], bits=bits, master=True)
    learn.adamw_step([before], [g], step=1, **other)
    assert torch.equal(p, before)
    for k in names:
        assert torch.equal(moved[k].view(torch.uint8), other[k].view(torch.uint8))
