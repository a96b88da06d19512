"""Operators of a policy trained over the environments and expansions of ``mymyr_b200.rl``, as CUDA kernels over torch
tensors: ``embedding`` (token embeddings and their gradient), ``logprobs`` (log-probabilities of given tokens or
actions, with entropy and the best alternatives, and their gradient) and the AdamW step over all of a policy's tensors
at once (``AdamW``, ``adamw_step``). The first two take part in torch's autograd.

Work runs on the tensors' device, on torch's current stream there or on the raw stream handle ``stream``, and is
asynchronous. Statistics and sums are 32-bit whatever the tensors' type (float32, bfloat16 or float16)."""

from __future__ import annotations

import array
import contextlib
import ctypes as C
import math
from dataclasses import dataclass

import torch
from torch.autograd.function import once_differentiable

from . import _lib
from ._lib import check, lib
from .task import default_context

_DTYPE = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
_BITS = {torch.int32: 32, torch.int64: 64}
BLOCK = _lib.B2_MOMENT_BLOCK
TOP_MAX = _lib.B2_TOP_MAX


def _ptr(t):
    return None if t is None else t.data_ptr()


def _context(t):
    return default_context(t.device.index).handle


def _stream(t):
    """The handle of torch's current stream on t's device (its stream object takes microseconds to make)."""
    return torch._C._cuda_getCurrentRawStream(t.device.index)


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


def _floating(t, what):
    if not isinstance(t, torch.Tensor) or not t.is_cuda or t.dtype not in _DTYPE:
        raise ValueError(f"{what} must be a CUDA tensor of float32, bfloat16 or float16")


def _indices(t, device, what):
    if not isinstance(t, torch.Tensor) or t.device != device or t.dtype not in _BITS:
        raise ValueError(f"{what} must be an int32 or int64 tensor on {device}")


# ------------------------------------------------------------------------------------------------ log-probabilities

@dataclass
class LogProbs:
    """What ``logprobs`` returns; every tensor float32 of the rows' shape but top_tokens (int64)."""

    logprob: torch.Tensor | None       # [...]: of each row's token (None without tokens)
    entropy: torch.Tensor              # [...]
    top_logprobs: torch.Tensor | None  # [..., top], from the best down; not differentiable
    top_tokens: torch.Tensor | None    # [..., top]; -1 past the row's tokens


def _logprobs_args(logits, tokens, offsets, mask, temperature, top):
    """logits [rows, width] with unit column stride, or ragged [width] with offsets."""
    a = _lib.LogprobsArgs()
    a.logits = logits.data_ptr()
    a.dtype = _DTYPE[logits.dtype]
    if offsets is None:
        a.rows, a.width = logits.shape
        a.row_stride = logits.stride(0)
    else:
        a.rows, a.width = offsets.numel() - 1, logits.numel()
        a.offsets = offsets.data_ptr()
        a.offsets_bits = _BITS[offsets.dtype]
    if tokens is not None:
        a.tokens = tokens.data_ptr()
        a.token_bits = _BITS[tokens.dtype]
    if mask is not None:
        a.mask = mask.data_ptr()
        a.mask_stride = mask.stride(0) if offsets is None else 0
    a.temperature = temperature
    a.top = top
    return a


def _logprobs_forward(logits, tokens, offsets, mask, temperature, top, stats=False):
    a = _logprobs_args(logits, tokens, offsets, mask, temperature, top)
    rows, dev = a.rows, logits.device
    entropy = torch.empty(rows, dtype=torch.float32, device=dev)
    a.entropy = entropy.data_ptr()
    logprob = top_logprobs = top_tokens = None
    if tokens is not None:
        logprob = torch.empty(rows, dtype=torch.float32, device=dev)
        a.logprob = logprob.data_ptr()
    if top:
        top_logprobs = torch.empty((rows, top), dtype=torch.float32, device=dev)
        top_tokens = torch.empty((rows, top), dtype=torch.int64, device=dev)
        a.top_logprobs, a.top_tokens = top_logprobs.data_ptr(), top_tokens.data_ptr()
    if stats:
        stats = torch.empty((rows, 4), dtype=torch.float32, device=dev)
        a.stats = stats.data_ptr()
    check(lib().b2_logprobs(_context(logits), C.byref(a), _stream(logits)))
    return a, stats, logprob, entropy, top_logprobs, top_tokens


class _LogProbs(torch.autograd.Function):
    @staticmethod
    def forward(ctx, logits, tokens, offsets, mask, temperature, top):
        ctx.args, stats, *out = _logprobs_forward(logits, tokens, offsets, mask, temperature, top, True)
        ctx.save_for_backward(logits, tokens, offsets, mask, stats)
        ctx.set_materialize_grads(False)
        if top:
            ctx.mark_non_differentiable(*out[2:])
        return tuple(out)

    @staticmethod
    @once_differentiable
    def backward(ctx, grad_logprob, grad_entropy, *_):
        logits, tokens, offsets, mask, stats = ctx.saved_tensors  # raises where one was changed in place since
        grad_logprob = None if grad_logprob is None else grad_logprob.contiguous()
        grad_entropy = None if grad_entropy is None else grad_entropy.contiguous()
        grad = torch.empty_like(logits, memory_format=torch.contiguous_format)
        a = ctx.args
        check(lib().b2_logprobs_backward(_context(logits), C.byref(a), _ptr(grad_logprob), _ptr(grad_entropy), grad.data_ptr(),
                                         a.width, _stream(logits)))
        return grad, None, None, None, None, None


def logprobs(logits: torch.Tensor, tokens: torch.Tensor | None = None, *, offsets: torch.Tensor | None = None,
             mask: torch.Tensor | None = None, temperature: float = 1.0, top: int = 0, stream=None) -> LogProbs:
    """Log-probabilities under softmax(logits / temperature): of each row's token, the entropy, and the ``top`` (at most
    32) best alternatives in order, equal logits by the lower index.

    ``logits`` [..., V] with ``tokens`` [...]; or, with ``offsets`` [N + 1], a vector of all rows' logits with row r at
    offsets[r] .. offsets[r + 1] (the successors of ``rl.expand``) and ``tokens`` [N] counted within the row, as an
    action of ``rl.BatchedEnv.step`` is. ``mask`` (bool, True: allowed) has the logits' shape or broadcasts to it.

    A negative token is no token (log-probability 0, no gradient); a masked one, or any token of a row that leaves
    nothing, has -inf; one past the row gives NaN. Such a row has entropy 0, no alternatives and a zero gradient."""
    _floating(logits, "logprobs: logits")
    dev = logits.device
    temperature = float(temperature)
    if not (temperature > 0.0 and math.isfinite(temperature)):
        raise ValueError("logprobs: temperature must be positive and finite")
    if not 0 <= int(top) <= TOP_MAX:
        raise ValueError(f"logprobs: top must be between 0 and {TOP_MAX}")
    top = int(top)
    if offsets is None:
        if logits.dim() < 1:
            raise ValueError("logprobs: logits must have a dimension of tokens")
        shape = logits.shape[:-1]
    else:
        _indices(offsets, dev, "logprobs: offsets")
        if logits.dim() != 1 or offsets.dim() != 1 or offsets.numel() < 1:
            raise ValueError("logprobs: with offsets [N + 1], logits must be the rows' one vector")
        shape = torch.Size((offsets.numel() - 1,))
        offsets = offsets.contiguous()
    if tokens is not None:
        _indices(tokens, dev, "logprobs: tokens")
        if tokens.shape != shape:
            raise ValueError(f"logprobs: tokens must have the rows' shape {tuple(shape)}, not {tuple(tokens.shape)}")
    if mask is not None and (not isinstance(mask, torch.Tensor) or mask.device != dev or mask.dtype != torch.bool):
        raise ValueError(f"logprobs: mask must be a bool tensor on {dev}")
    if stream is not None:
        with _on(stream, logits, tokens, offsets, mask):
            return logprobs(logits, tokens, offsets=offsets, mask=mask, temperature=temperature, top=top)
    if mask is not None:
        if offsets is None and mask.dim() == 1:
            mask = mask.expand(logits.shape[-1]).expand(shape.numel(), logits.shape[-1])
        elif mask.dim() <= logits.dim():
            mask = mask.expand(logits.shape)
            mask = mask.reshape(shape.numel(), logits.shape[-1]) if offsets is None else mask.contiguous()
        else:
            raise ValueError("logprobs: mask does not broadcast to the logits")
        if mask.stride(-1) != 1 and mask.shape[-1] > 1:
            mask = mask.contiguous()
    if logits.dim() > 2 or (logits.dim() == 1 and offsets is None):
        logits = logits.reshape(shape.numel(), logits.shape[-1])
    if logits.stride(-1) != 1 and logits.shape[-1] > 1:
        logits = logits.contiguous()
    if tokens is not None:
        tokens = tokens.reshape(-1).contiguous()
    if logits.requires_grad and torch.is_grad_enabled():
        logprob, entropy, top_logprobs, top_tokens = _LogProbs.apply(logits, tokens, offsets, mask, temperature, top)
    else:
        _, _, logprob, entropy, top_logprobs, top_tokens = _logprobs_forward(logits, tokens, offsets, mask,
                                                                             temperature, top)
    if len(shape) != 1:
        entropy = entropy.view(shape)
        logprob = None if logprob is None else logprob.view(shape)
        if top:
            top_logprobs, top_tokens = top_logprobs.view(*shape, top), top_tokens.view(*shape, top)
    return LogProbs(logprob, entropy, top_logprobs, top_tokens)


# ------------------------------------------------------------------------------------------------ embeddings

def _embedding_args(tokens, weight_shape, dtype, scale):
    a = _lib.EmbeddingArgs()
    a.tokens = tokens.data_ptr()
    a.token_bits = _BITS[tokens.dtype]
    a.dtype = _DTYPE[dtype]
    a.count = tokens.numel()
    a.vocabulary, a.width = weight_shape
    a.scale = scale
    return a


def _embedding_forward(tokens, weight, scale):
    a = _embedding_args(tokens, weight.shape, weight.dtype, scale)
    rows = torch.empty((a.count, a.width), dtype=weight.dtype, device=weight.device)
    check(lib().b2_embedding(_context(weight), C.byref(a), weight.data_ptr(), weight.stride(0), rows.data_ptr(),
                             _stream(weight)))
    return a, rows


class _Embedding(torch.autograd.Function):
    @staticmethod
    def forward(ctx, tokens, weight, scale):
        ctx.args, rows = _embedding_forward(tokens, weight, scale)
        ctx.save_for_backward(tokens)
        return rows

    @staticmethod
    @once_differentiable
    def backward(ctx, grad):
        a = ctx.args
        tokens, = ctx.saved_tensors
        if grad.stride(1) != 1 and grad.shape[1] > 1:
            grad = grad.contiguous()
        grad_weight = torch.empty((a.vocabulary, a.width), dtype=grad.dtype, device=grad.device)
        size = lib().b2_embedding_workspace(C.byref(a))
        workspace = torch.empty(size, dtype=torch.uint8, device=grad.device)
        check(lib().b2_embedding_backward(_context(grad), C.byref(a), grad.data_ptr(), grad.stride(0),
                                          grad_weight.data_ptr(), workspace.data_ptr(), size, _stream(grad)))
        return None, grad_weight, None


def embedding(tokens: torch.Tensor, weight: torch.Tensor, *, scale: float = 1.0, stream=None) -> torch.Tensor:
    """scale * weight[tokens], [..., D] for tokens [...] and weight [V, D]. A negative token is an empty place (a row of
    zeros, no gradient), one past the table gives a row of NaN. The gradient of the table sums each token's rows in
    32 bits and in the same order on every call."""
    _floating(weight, "embedding: weight")
    if weight.dim() != 2:
        raise ValueError("embedding: weight must be [V, D]")
    _indices(tokens, weight.device, "embedding: tokens")
    if stream is not None:
        with _on(stream, tokens, weight):
            return embedding(tokens, weight, scale=scale)
    shape = tokens.shape
    tokens = tokens.reshape(-1).contiguous()
    if weight.stride(1) != 1 and weight.shape[1] > 1:
        weight = weight.contiguous()
    if weight.requires_grad and torch.is_grad_enabled():
        rows = _Embedding.apply(tokens, weight, float(scale))
    else:
        _, rows = _embedding_forward(tokens, weight, float(scale))
    return rows if len(shape) == 1 else rows.view(*shape, weight.shape[1])


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
    for p in params:
        _floating(p, "adamw_state: a parameter")
    dev = params[0].device
    blocks = sum(_blocks(p.numel()) for p in params)
    dtype = torch.float32 if bits == 32 else torch.float8_e4m3fn
    state = {k: torch.zeros(blocks * BLOCK, dtype=torch.float32, device=dev).to(dtype) for k in
             ("exp_avg", "exp_avg_sq")}
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
    """One AdamW update of all ``params`` (contiguous, of any sizes) in place, with the moments of ``adamw_state``:

        m = b1 m + (1 - b1) g;  v = b2 v + (1 - b2) g^2
        p = p (1 - lr weight_decay) - lr (m / (1 - b1^step)) / (sqrt(v / (1 - b2^step)) + eps)

    A gradient is of its parameter's type or float32; one that is None leaves its tensor alone. Parameters of 16 bits
    are rounded to nearest from ``master`` if given. 8-bit moments are rounded for storage only: the first to nearest,
    the second to one of its two neighbours by random numbers of (``seed``, step, element), so that the small steps of
    a slow average are kept in the mean."""
    params, grads = list(params), list(grads)
    if len(params) != len(grads):
        raise ValueError("adamw_step: one gradient for each parameter")
    if not isinstance(exp_avg, torch.Tensor) or not exp_avg.is_cuda:
        raise ValueError("adamw_step: the moments must be CUDA tensors")
    dev, bits = exp_avg.device, 32 if exp_avg.dtype == torch.float32 else 8
    if stream is not None:
        with _on(stream, exp_avg, exp_avg_sq, exp_avg_scale, exp_avg_sq_scale, master, *params, *grads):
            return adamw_step(params, grads, exp_avg, exp_avg_sq, step=step, lr=lr, betas=betas, eps=eps,
                              weight_decay=weight_decay, exp_avg_scale=exp_avg_scale,
                              exp_avg_sq_scale=exp_avg_sq_scale, master=master, seed=seed)
    elements = exp_avg.numel()
    blocks = elements // BLOCK
    kind = torch.float32 if bits == 32 else torch.float8_e4m3fn
    for t, dtype, n, name in ((exp_avg, kind, elements, "exp_avg"), (exp_avg_sq, kind, elements, "exp_avg_sq"),
                              (exp_avg_scale, torch.float32, blocks, "exp_avg_scale"),
                              (exp_avg_sq_scale, torch.float32, blocks, "exp_avg_sq_scale"),
                              (master, torch.float32, elements, "master")):
        if t is None:
            if name == "master" or (bits == 32 and name.endswith("scale")):
                continue
            raise ValueError(f"adamw_step: 8-bit moments need {name}")
        if t.dtype != dtype or t.device != dev or t.numel() != n or not t.is_contiguous():
            raise ValueError(f"adamw_step: {name} must be a contiguous {dtype} tensor of {n} elements on {dev}")
    step = int(step)
    if step < 1:
        raise ValueError("adamw_step: step counts from 1")
    sizes = [p.numel() for p in params]
    places, at = [], 0
    for n in sizes:
        places.append(at)
        at += -(-n // BLOCK)
    if at != blocks or elements % BLOCK:
        raise ValueError(f"adamw_step: the moments must hold {at} blocks of {BLOCK} elements, not {elements} elements")
    if 0 in sizes or any(g is None for g in grads):
        kept = [i for i, g in enumerate(grads) if g is not None and sizes[i]]
        live, grads = [params[i] for i in kept], [grads[i] for i in kept]
        sizes, places = [sizes[i] for i in kept], [places[i] for i in kept]
    else:
        live = params
    if not live:
        return
    index = dev.index
    if {t.get_device() for t in live} | {t.get_device() for t in grads} != {index}:
        raise ValueError(f"adamw_step: parameters and gradients must be on {dev}")
    if not all([p.is_contiguous() for p in live]):
        raise ValueError("adamw_step: parameters must be contiguous")
    if [g.numel() for g in grads] != sizes:
        raise ValueError("adamw_step: a gradient has its parameter's shape")
    if not all([g.is_contiguous() for g in grads]):
        grads = [g.contiguous() for g in grads]
    dtypes = [(p.dtype, g.dtype) for p, g in zip(live, grads)]
    kinds = set(dtypes)
    for p, g in kinds:
        if p not in _DTYPE or (g != p and g != torch.float32):
            raise ValueError("adamw_step: parameters are float32, bfloat16 or float16, a gradient of its parameter's "
                             "type or float32")
    a = _lib.AdamwArgs()
    a.moment_bits, a.blocks = bits, blocks
    a.exp_avg, a.exp_avg_sq = exp_avg.data_ptr(), exp_avg_sq.data_ptr()
    if bits == 8:
        a.exp_avg_scale, a.exp_avg_sq_scale = exp_avg_scale.data_ptr(), exp_avg_sq_scale.data_ptr()
    a.master = _ptr(master)
    a.lr, (a.beta1, a.beta2), a.eps, a.weight_decay = lr, betas, eps, weight_decay
    a.step, a.seed = step, int(seed) & 0xFFFFFFFF
    rows = zip(live, grads, sizes, places)
    for kind in kinds:  # one launch for each
        mine = rows if len(kinds) == 1 else [r for r, k in zip(zip(live, grads, sizes, places), dtypes) if k == kind]
        # the fields of b2_adamw_tensor, as four words
        table = array.array("Q", [x for p, g, n, b in mine for x in (p.data_ptr(), g.data_ptr(), n, b)])
        a.tensors, a.count = table.buffer_info()[0], len(table) // 4
        a.param_dtype, a.grad_dtype = _DTYPE[kind[0]], _DTYPE[kind[1]]
        check(lib().b2_adamw(_context(exp_avg), C.byref(a), _stream(exp_avg)))
    torch.autograd.graph.increment_version(live)


class AdamW:
    """AdamW over a policy's parameters, all of a group's tensors in one launch (``adamw_step``). ``params``: tensors,
    or groups as dicts with "params" and their own lr, betas, eps or weight_decay. ``bits``: 32 or 8 for the moments;
    ``master``: 32-bit copies of 16-bit parameters. Each group keeps its moments in flat tensors of its own."""

    def __init__(self, params, lr: float = 1e-3, betas: tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, *, bits: int = 32, master: bool = False, seed: int = 0):
        defaults = {"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay}
        params = list(params)
        groups = params if params and isinstance(params[0], dict) else [{"params": params}]
        self.param_groups = [defaults | g | {"params": list(g["params"])} for g in groups]
        self.steps = 0
        self.seed = int(seed)
        self.state = [adamw_state(g["params"], bits=bits, master=master) for g in self.param_groups]

    def zero_grad(self) -> None:
        """Drops the parameters' gradients."""
        for g in self.param_groups:
            for p in g["params"]:
                p.grad = None

    def step(self, stream=None) -> None:
        """Updates every parameter that has a gradient."""
        self.steps += 1
        with torch.no_grad():
            for i, (g, s) in enumerate(zip(self.param_groups, self.state)):
                adamw_step(g["params"], [p.grad for p in g["params"]], step=self.steps, lr=g["lr"], betas=g["betas"],
                           eps=g["eps"], weight_decay=g["weight_decay"], seed=self.seed + i, stream=stream, **s)

    def state_dict(self) -> dict:
        """The step count, the groups' options and their moments (the tensors themselves, not copies)."""
        return {"steps": self.steps, "seed": self.seed, "state": self.state,
                "groups": [{k: v for k, v in g.items() if k != "params"} for g in self.param_groups]}

    def load_state_dict(self, state: dict) -> None:
        """Takes over what state_dict() gave for an optimizer over tensors of the same sizes."""
        if len(state["state"]) != len(self.state):
            raise ValueError("AdamW: another number of groups")
        for mine, given in zip(self.state, state["state"]):
            if mine.keys() != given.keys() or any(mine[k].shape != given[k].shape or mine[k].dtype != given[k].dtype
                                                  for k in mine):
                raise ValueError("AdamW: moments of other sizes or types")
        for mine, given in zip(self.state, state["state"]):
            for k in mine:
                mine[k].copy_(given[k])
        for g, options in zip(self.param_groups, state["groups"]):
            g.update(options)
        self.steps, self.seed = int(state["steps"]), int(state["seed"])
