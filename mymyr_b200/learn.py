"""Operators of a policy trained over the environments and expansions of ``mymyr_b200.rl``, as CUDA kernels over torch
tensors: ``embedding`` (token embeddings and their gradient), ``logprobs`` (log-probabilities of given tokens or
actions, with entropy and the best alternatives, and their gradient) and the AdamW step over all of a policy's tensors
at once (``AdamW``, ``adamw_step``). The first two take part in torch's autograd.

Work runs on the tensors' device, on torch's current stream there or on the raw stream handle ``stream``, and is
asynchronous. All but the AdamW step can be captured in CUDA graphs. Statistics and sums are 32-bit whatever the
tensors' type (float32, bfloat16 or float16)."""

from __future__ import annotations

import contextlib
import importlib.machinery
import importlib.util
from dataclasses import dataclass

import torch

from . import _lib
from ._lib import LIB_PATH, lib

BLOCK = _lib.B2_MOMENT_BLOCK
TOP_MAX = _lib.B2_TOP_MAX
_FLOATS = (torch.float32, torch.bfloat16, torch.float16)


def _load():
    """The torch module of these operators (csrc/torch_learn.cpp); raises if it was not built."""
    path = LIB_PATH.with_name("_learn.so")
    if not path.exists():
        raise RuntimeError(f"mymyr_b200: {path} is missing; build it with __graft_entry__.build() "
                           "(there is no CPU fallback)")
    lib()  # it calls this library
    loader = importlib.machinery.ExtensionFileLoader("_learn", str(path))
    module = importlib.util.module_from_spec(importlib.util.spec_from_loader("_learn", loader))
    loader.exec_module(module)
    return module


_learn = _load()


@contextlib.contextmanager
def _on(stream, *tensors):
    """The raw stream as torch's current one: what a call allocates belongs to it, and the inputs' memory is kept until
    it is done with them."""
    device = tensors[0].device
    s = torch.cuda.ExternalStream(stream, device=device)
    with torch.cuda.stream(s):
        yield
        for t in tensors:
            if t is not None:
                t.record_stream(s)


# ------------------------------------------------------------------------------------------------ log-probabilities

@dataclass
class LogProbs:
    """What ``logprobs`` returns; every tensor float32 of the rows' shape but top_tokens (int64)."""

    logprob: torch.Tensor | None       # [...]: of each row's token (None without tokens)
    entropy: torch.Tensor              # [...]
    top_logprobs: torch.Tensor | None  # [..., top], from the best down; not differentiable
    top_tokens: torch.Tensor | None    # [..., top]; -1 past the row's tokens


def logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, offsets: torch.Tensor | None = None,
             mask: torch.Tensor | None = None, temperature: float = 1.0, top: int = 0, stream=None) -> LogProbs:
    """Log-probabilities under softmax(logits / temperature): of each row's token, the entropy, and the ``top`` (at most
    32) best alternatives in order, equal logits by the lower index.

    ``logits`` [..., V] with ``tokens`` [...]; or, with ``offsets`` [N + 1], a vector of all rows' logits with row r at
    offsets[r] .. offsets[r + 1] (the successors of ``rl.expand``) and ``tokens`` [N] counted within the row, as an
    action of ``rl.BatchedEnv.step`` is (for a gradient, offsets must not decrease: overlapping rows would overwrite one
    another). ``mask`` (bool, True: allowed) has the logits' shape or broadcasts to it.

    A negative token is no token (log-probability 0, no gradient); a masked one, or any token of a row that leaves
    nothing, has -inf; one past the row gives NaN. A row that leaves nothing has entropy 0, no alternatives and a zero
    gradient."""
    if stream is not None:
        with _on(stream, logits, tokens, offsets, mask):
            return LogProbs(*_learn.logprobs(logits, tokens, offsets, mask, temperature, top))
    return LogProbs(*_learn.logprobs(logits, tokens, offsets, mask, temperature, top))


# ------------------------------------------------------------------------------------------------ embeddings

def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, stream=None) -> torch.Tensor:
    """scale * weight[tokens], [..., D] for tokens [...] and weight [V, D]. A negative token is an empty place (a row of
    zeros, no gradient), one past the table gives a row of NaN. The gradient of the table sums each token's rows in
    32 bits and in the same order on every call."""
    if stream is not None:
        with _on(stream, weight, tokens):
            return _learn.embedding(tokens, weight, scale)
    return _learn.embedding(tokens, weight, scale)


# ------------------------------------------------------------------------------------------------ AdamW

def _blocks(elements: int) -> int:
    return -(-elements // BLOCK)


def adamw_state(params, *, bits: int = 32, master: bool = False) -> dict[str, torch.Tensor]:
    """Fresh moments for ``adamw_step`` over ``params``, as its keyword arguments: ``exp_avg`` and ``exp_avg_sq`` hold
    the tensors one after the other, each from a block of 256 elements of its own. ``bits=8``: float8_e4m3fn codes with
    a float32 scale for each block; exp_avg_sq then holds the square root. ``master``: 32-bit copies of the parameters
    in the same layout, for parameters of 16 bits."""
    params = list(params)
    if bits not in (32, 8):
        raise ValueError("adamw_state: bits must be 32 or 8")
    if not params:
        raise ValueError("adamw_state: no parameters")
    if any(not p.is_cuda or p.dtype not in _FLOATS for p in params):
        raise ValueError("adamw_state: parameters must be CUDA tensors of float32, bfloat16 or float16")
    dev = params[0].device
    blocks = sum(_blocks(p.numel()) for p in params)
    zeros = [torch.zeros(blocks * BLOCK, dtype=torch.float32 if bits == 32 else torch.uint8, device=dev)
             for _ in range(2)]
    state = dict(zip(("exp_avg", "exp_avg_sq"), zeros if bits == 32 else [z.view(torch.float8_e4m3fn) for z in zeros]))
    if bits == 8:
        state |= {k: torch.ones(blocks, dtype=torch.float32, device=dev) for k in
                  ("exp_avg_scale", "exp_avg_sq_scale")}
    if master:
        state["master"] = torch.zeros(blocks * BLOCK, dtype=torch.float32, device=dev)
        at = 0
        for p in params:
            state["master"][at:at + p.numel()] = p.detach().reshape(-1)
            at += _blocks(p.numel()) * BLOCK
    return state


def adamw_step(params, grads, exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor, *, step: int, lr: float = 1e-3,
               betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
               exp_avg_scale: torch.Tensor | None = None, exp_avg_sq_scale: torch.Tensor | None = None,
               master: torch.Tensor | None = None, seed: int = 0, stream=None) -> None:
    """One AdamW update of all ``params`` (contiguous, of any sizes, none overlapping) in place, with the moments of
    ``adamw_state``:

        m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
        p = p (1 - lr weight_decay) - lr (m / (1 - b1^step)) / (sqrt(v / (1 - b2^step)) + eps)

    Moments of another origin (a part of a larger buffer) must be contiguous and start on a boundary of eight elements.
    A gradient is of its parameter's type or float32; one that is None leaves its tensor alone. Parameters of 16 bits
    are rounded to nearest from ``master`` if given. 8-bit moments are rounded for storage only: the first to nearest,
    the second to one of its two neighbours by random numbers of (``seed``, step, element), so that the small steps of
    a slow average are kept in the mean.

    A CUDA graph would repeat one step's corrections and random numbers: a call on a stream under capture is refused."""
    params, grads = list(params), list(grads)
    with contextlib.nullcontext() if stream is None else _on(stream, exp_avg, exp_avg_sq, exp_avg_scale,
                                                            exp_avg_sq_scale, master, *params, *grads):
        _learn.adamw_step(params, grads, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, master, step, lr,
                          *betas, eps, weight_decay, seed & 0xFFFFFFFF)


class AdamW:
    """AdamW over a policy's parameters, all of a group's tensors in one launch (``adamw_step``). ``params``: tensors,
    or groups as dicts with "params" and their own lr, betas, eps or weight_decay. ``bits``: 32 or 8 for the moments;
    ``master``: 32-bit copies of 16-bit parameters. Each group keeps its moments in flat tensors of its own. A parameter's
    step number, by which its averages are corrected, counts the steps that it had a gradient for; where a group's differ
    (some had none at times), each number is a launch."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, bits: int = 32, master: bool = False, seed: int = 0):
        defaults = {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay}
        if isinstance(params, torch.Tensor):  # its rows would be tensors without gradients
            raise ValueError("AdamW: params must be a list of tensors or of groups")
        params = list(params)
        groups = params if params and isinstance(params[0], dict) else [{"params": params}]
        self.param_groups = [defaults | g | {"params": [p] if isinstance(p := g["params"], torch.Tensor) else list(p)}
                             for g in groups]
        every = [id(p) for g in self.param_groups for p in g["params"]]
        if len(set(every)) < len(every):  # two threads would update the same numbers at once
            raise ValueError("AdamW: a parameter is given twice")
        self.steps = 0
        self.param_steps = [[0] * len(g["params"]) for g in self.param_groups]
        self.seed = int(seed)
        self.state = [adamw_state(g["params"], bits=bits, master=master) for g in self.param_groups]

    def zero_grad(self) -> None:
        """Drops the parameters' gradients."""
        for g in self.param_groups:
            for p in g["params"]:
                p.grad = None

    def step(self, stream=None) -> None:
        """Updates every parameter that has a gradient."""
        with torch.no_grad():
            for i, (g, s, counts) in enumerate(zip(self.param_groups, self.state, self.param_steps)):
                grads = [p.grad for p in g["params"]]
                now = [n if x is None else n + 1 for n, x in zip(counts, grads)]
                for step in sorted({n for n, x in zip(now, grads) if x is not None}):
                    adamw_step(g["params"], [x if n == step else None for n, x in zip(now, grads)], step=step, lr=g["lr"],
                               betas=g["betas"], eps=g["eps"], weight_decay=g["weight_decay"], seed=self.seed + i,
                               stream=stream, **s)
                counts[:] = now
        self.steps += 1

    def state_dict(self) -> dict:
        """The step counts, the groups' options and their moments (the tensors themselves, not copies)."""
        return {"steps": self.steps, "param_steps": [list(c) for c in self.param_steps], "seed": self.seed,
                "state": self.state,
                "groups": [{k: v for k, v in g.items() if k != "params"} for g in self.param_groups]}

    def load_state_dict(self, state: dict) -> None:
        """Takes over what state_dict() gave for an optimizer over tensors of the same sizes."""
        if len(state["state"]) != len(self.state):
            raise ValueError("AdamW: another number of groups")
        for mine, given in zip(self.state, state["state"]):
            if mine.keys() != given.keys() or any(mine[k].shape != given[k].shape or mine[k].dtype != given[k].dtype
                                                  for k in mine):
                raise ValueError("AdamW: moments of other sizes or types")
        # without counts of their own (of an earlier version) all parameters are at the optimizer's step
        counts = state.get("param_steps") or [[int(state["steps"])] * len(c) for c in self.param_steps]
        if [len(c) for c in counts] != [len(c) for c in self.param_steps]:
            raise ValueError("AdamW: another number of parameters")
        for mine, given in zip(self.state, state["state"]):
            for k in mine:
                mine[k].copy_(given[k])
        for g, options in zip(self.param_groups, state["groups"]):
            g.update(options)
        self.steps, self.seed = int(state["steps"]), int(state["seed"])
        self.param_steps = [[int(n) for n in c] for c in counts]
