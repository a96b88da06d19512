"""The learner's operators (``mymyr_b200.learn``): what is measured, and their plain forms.

Three operators make a policy's training step over batched environments and its scoring in use: the lookup of token
embeddings with its gradient, the log-probabilities of given tokens (actions) with entropy and the best alternatives
and their gradient, and the AdamW step over all of a policy's tensors with moments in 32 or in 8 bits.

``run`` computes them in elementary torch operations in 32 bits, or with the package's kernels where ``own`` is set.
"""

import math

import torch

own = False

DEVICE = "cuda"
TYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
BLOCK = 256  # elements of a moment block: one scale each in the 8-bit form, and the unit of a tensor's place in 32 bits
INF = float("inf")


# ------------------------------------------------------------------------------------------------ cases

def _logprobs(rows, width, dtype, *, train, top, masked=False, temperature=1.0):
    return {"op": "logprobs", "rows": rows, "width": width, "dtype": dtype, "train": train, "top": top,
            "masked": masked, "temperature": temperature, "ragged": False}


def _actions(rows, least, most, dtype, *, train, top):
    return {"op": "logprobs", "rows": rows, "width": most, "least": least, "dtype": dtype, "train": train, "top": top,
            "masked": False, "temperature": 1.0, "ragged": True}


def _embedding(tokens, vocabulary, width, dtype, *, train, skew, empty):
    return {"op": "embedding", "tokens": tokens, "vocabulary": vocabulary, "width": width, "dtype": dtype,
            "train": train, "skew": skew, "empty": empty}


def _adamw(layers, width, extra, dtype, *, bits, master):
    return {"op": "adamw", "layers": layers, "width": width, "extra": extra, "dtype": dtype, "bits": bits,
            "master": master}


def listed():
    return [
        # serving: one sequence's next token, its twenty best alternatives
        dict(_logprobs(1, 131072, "bf16", train=False, top=20, temperature=0.7), name="one row"),
        # serving: a small batch under a grammar's mask, a vocabulary of odd size; some rows have no token left
        dict(_logprobs(24, 100003, "f16", train=False, top=5, masked=True), name="few masked rows"),
        # scoring a batch of rollouts with their alternatives
        dict(_logprobs(2048, 50001, "f32", train=False, top=8), name="scored rollouts"),
        # a training batch: log-probability and entropy of each token, and the gradient of the logits
        dict(_logprobs(8192, 65536, "bf16", train=True, top=0), name="trained tokens"),
        # the applicable actions of 65,536 sliding-tile environments (2 to 4 each)
        dict(_actions(65536, 2, 4, "f32", train=True, top=0), name="tile actions"),
        # the applicable actions of a large lifted task: none (a dead end) to a thousand for each state
        dict(_actions(8192, 0, 1000, "bf16", train=True, top=4), name="many actions"),
        # serving: the next tokens of eight sequences
        dict(_embedding(8, 131072, 2048, "bf16", train=False, skew=1.0, empty=0.0), name="next tokens"),
        # 2,048 states of 10,560 atoms at 5 % density: each true atom a token, every row of the table hit often
        dict(_embedding(2048 * 528, 10560, 128, "f32", train=True, skew=1.0, empty=0.02), name="state atoms"),
        # a training batch of text: few frequent tokens, many rare ones, padding; most of the table untouched
        dict(_embedding(16383, 65536, 1024, "bf16", train=True, skew=4.0, empty=0.05), name="text tokens"),
        # a small policy network in full precision
        dict(_adamw(4, 256, 257, "f32", bits=32, master=False), name="small policy"),
        # a 170M-parameter model in bf16 with 32-bit masters and moments
        dict(_adamw(16, 1024, 5003, "bf16", bits=32, master=True), name="moments in 32 bits"),
        # a 330M-parameter model in bf16 with 8-bit moments
        dict(_adamw(16, 1408, 8191, "bf16", bits=8, master=False), name="moments in 8 bits"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["dense", "dense", "ragged", "embedding", "embedding", "adamw"])
    dtype = rng.choice(["f32", "bf16", "f16"])
    train = rng.random() < 0.5
    if kind == "dense":
        width = _log_int(rng, 2, 262144)
        rows = _log_int(rng, 1, max(1, min(65536, 2 ** 27 // width)))
        return _logprobs(rows, width, dtype, train=train, top=rng.choice([0, 1, 5, 20, 32]),
                         masked=rng.random() < 0.4, temperature=rng.choice([1.0, 0.7, 1.3]))
    if kind == "ragged":
        most = _log_int(rng, 2, 5000)
        rows = _log_int(rng, 1, max(1, min(131072, 2 ** 26 // most)))
        return _actions(rows, rng.choice([0, 1]), most, dtype, train=train, top=rng.choice([0, 1, 4, 16]))
    if kind == "embedding":
        width = _log_int(rng, 1, 8192)
        vocabulary = _log_int(rng, 2, min(262144, 2 ** 28 // width))
        tokens = _log_int(rng, 1, min(2 ** 20, 2 ** 28 // width))
        return _embedding(tokens, vocabulary, width, dtype, train=train, skew=rng.choice([1.0, 2.0, 4.0]),
                          empty=rng.choice([0.0, 0.1]))
    width = _log_int(rng, 8, 1024)
    layers = rng.randint(1, 16)
    return _adamw(layers, width, _log_int(rng, 1, 5003), dtype, bits=rng.choice([32, 8]),
                  master=dtype != "f32" and rng.random() < 0.5)


# ------------------------------------------------------------------------------------------------ inputs

def _generator(seed):
    g = torch.Generator(device=DEVICE)
    g.manual_seed(int(seed))
    return g


def _prepare_logprobs(case, g):
    rows, width, dtype = case["rows"], case["width"], TYPES[case["dtype"]]
    s = {}
    if case["ragged"]:
        # counts towards the small end, as applicable actions are, and both ends among them; the seed orders them
        u = torch.arange(rows, device=DEVICE) / max(1, rows - 1)
        count = (case["least"] + u.double() ** 2 * (width - case["least"])).round().long()
        count = count[torch.randperm(rows, generator=g, device=DEVICE)]
        offsets = torch.zeros(rows + 1, dtype=torch.int32, device=DEVICE)
        offsets[1:] = count.cumsum(0)
        total = int(offsets[-1])
        logits = torch.randn(total, generator=g, device=DEVICE) * 2
        pick = (torch.rand(rows, generator=g, device=DEVICE) * count).long()
        tokens = torch.where(count > 0, torch.minimum(pick, count - 1), torch.full_like(pick, -1))
        s["offsets"] = offsets
    else:
        logits = torch.randn(rows, width, generator=g, device=DEVICE) * 2
        if case["masked"]:
            mask = torch.rand(rows, width, generator=g, device=DEVICE) < 0.3
            mask[rows // 2] = rows == 1  # a row with nothing left
            s["mask"] = mask
            best = logits.masked_fill(~mask, -INF).argmax(1)
        else:
            best = logits.argmax(1)
        other = torch.randint(0, width, (rows,), generator=g, device=DEVICE)
        if case["masked"]:
            other = torch.where(mask.gather(1, other[:, None])[:, 0], other, best)
        tokens = torch.where(torch.rand(rows, generator=g, device=DEVICE) < 0.5, best, other)
        tokens[rows // 3] = -1 if rows > 3 else tokens[rows // 3]  # a place without a token
    s["logits"] = logits.to(dtype).requires_grad_(case["train"])
    s["tokens"] = tokens
    if case["train"]:
        s["grad_logprob"] = torch.randn(rows, generator=g, device=DEVICE) / rows
        s["grad_entropy"] = torch.randn(rows, generator=g, device=DEVICE) * (0.1 / rows)
    return s


def _prepare_embedding(case, g):
    n, vocabulary, width, dtype = case["tokens"], case["vocabulary"], case["width"], TYPES[case["dtype"]]
    u = torch.rand(n, generator=g, device=DEVICE)
    tokens = (u ** case["skew"] * vocabulary).long().clamp(0, vocabulary - 1)
    tokens = (tokens * 7919 + 13) % vocabulary if vocabulary % 7919 else tokens  # the frequent ones lie apart
    if case["empty"]:
        tokens[torch.rand(n, generator=g, device=DEVICE) < case["empty"]] = -1
    s = {"tokens": tokens}
    s["weight"] = (torch.randn(vocabulary, width, generator=g, device=DEVICE) * 0.02).to(dtype)
    s["weight"].requires_grad_(case["train"])
    if case["train"]:
        s["grad"] = (torch.randn(n, width, generator=g, device=DEVICE) * 1e-2).to(dtype)
    return s


def _shapes(case):
    """A network's tensors: for each layer two square matrices, a wide one, a bias (up to twelve layers); and a table of
    `extra` rows."""
    w = case["width"]
    each = [(w, w), (w, w), (w, 8 * w + 3), (w + 1,)][: 3 if case["layers"] > 12 else 4]
    return each * case["layers"] + [(case["extra"], w)]


def _spans(shapes):
    """Each tensor's place in the moments: [first element, elements], every tensor from a block of its own."""
    at, spans = 0, []
    for shape in shapes:
        n = math.prod(shape)
        spans.append((at, n))
        at += -(-n // BLOCK) * BLOCK
    return spans, at


def _prepare_adamw(case, g):
    dtype = TYPES[case["dtype"]]
    shapes = _shapes(case)
    spans, total = _spans(shapes)

    def normal(shape, scale):
        return torch.randn(*shape, generator=g, device=DEVICE) * scale

    s = {"step": 1000, "seed": int(torch.randint(0, 2 ** 31, (), generator=g, device=DEVICE)), "spans": spans, "total": total}
    full = [normal(shape, 0.02) for shape in shapes]
    s["params"] = [p.to(dtype) for p in full]
    # gradients of very different size from tensor to tensor, some elements without any
    s["grads"] = [(normal(shape, 10.0 ** -(2 + i % 4)) * (torch.rand(*shape, generator=g, device=DEVICE) > 0.1))
                  .to(dtype) for i, shape in enumerate(shapes)]
    held = torch.zeros(total, device=DEVICE)
    for x, (at, n) in zip(s["grads"], spans):
        held[at:at + n] = x.reshape(-1).float()
    m = held * 0.3
    r = held.abs() * 0.8
    if case["bits"] == 8:
        s["exp_avg"], s["exp_avg_scale"] = _first_8_bits(m)
        s["exp_avg_sq"], s["exp_avg_sq_scale"] = _second_8_bits(r, torch.full_like(r, 0.5))
    else:
        s["exp_avg"], s["exp_avg_sq"] = m, r * r
    if case["master"]:
        s["master"] = torch.zeros(total, device=DEVICE)
        for x, (at, n) in zip(full, spans):
            s["master"][at:at + n] = x.reshape(-1)
    return s


def prepare(case, seed):
    g = _generator(seed)
    s = {"logprobs": _prepare_logprobs, "embedding": _prepare_embedding, "adamw": _prepare_adamw}[case["op"]](case, g)
    s["case"] = case
    return s


# ------------------------------------------------------------------------------------------------ plain forms

def _plain_logprobs(s):
    case = s["case"]
    logits, tokens, rows, top = s["logits"].detach(), s["tokens"], case["rows"], case["top"]
    if case["ragged"]:
        offsets = s["offsets"].long()
        place = torch.arange(logits.numel(), device=DEVICE)
        row = torch.repeat_interleave(torch.arange(rows, device=DEVICE), offsets.diff(), output_size=logits.numel())
        place = place - offsets[row]
        x = torch.full((rows, case["width"]), -INF, device=DEVICE)
        x[row, place] = logits.float()
    else:
        x = logits.float()
        if "mask" in s:
            x = torch.where(s["mask"], x, -INF)
    best = x.amax(1, keepdim=True)
    dead = best == -INF
    d = (x - torch.where(dead, 0.0, best)) / case["temperature"]
    e = d.exp()
    total = e.sum(1, keepdim=True)
    log_total = total.log()
    log_p = torch.where(d == -INF, -INF, d - log_total)
    p = e / torch.where(dead, 1.0, total)
    finite = torch.where(d == -INF, 0.0, log_p)
    entropy = -(p * finite).sum(1)
    out = {"entropy": entropy}
    given = tokens >= 0
    at = tokens.clamp(min=0)[:, None]
    out["logprob"] = torch.where(given, log_p.gather(1, at)[:, 0], 0.0)
    if top:
        order = torch.sort(x, dim=1, descending=True, stable=True)
        k = min(top, x.shape[1])
        ids, values = order.indices[:, :k], log_p.gather(1, order.indices[:, :k])
        ids = torch.where(order.values[:, :k] == -INF, -1, ids)
        values = torch.where(ids < 0, -INF, values)
        out["top_tokens"] = torch.full((rows, top), -1, dtype=torch.int64, device=DEVICE)
        out["top_tokens"][:, :k] = ids
        out["top_logprobs"] = torch.full((rows, top), -INF, device=DEVICE)
        out["top_logprobs"][:, :k] = values
    if case["train"]:
        gl = torch.where(given, s["grad_logprob"], 0.0)[:, None]
        ge = s["grad_entropy"][:, None]
        grad = -p * (gl + ge * (finite + entropy[:, None]))
        grad.scatter_add_(1, at, torch.where(dead, 0.0, gl))
        grad /= case["temperature"]
        if "mask" in s:
            grad = torch.where(s["mask"], grad, 0.0)
        out["grad"] = (grad[row, place] if case["ragged"] else grad).to(logits.dtype)
    return out


def _scale(case):
    return math.sqrt(case["width"])


def _plain_embedding(s):
    tokens, weight, scale = s["tokens"], s["weight"].detach(), _scale(s["case"])
    empty = (tokens < 0)[:, None]
    at = tokens.clamp(min=0)
    out = {"rows": torch.where(empty, 0.0, weight[at].float() * scale).to(weight.dtype)}
    if s["case"]["train"]:
        grad = torch.zeros(weight.shape, device=DEVICE)
        grad.index_add_(0, at, torch.where(empty, 0.0, s["grad"].float()))
        out["grad"] = (grad * scale).to(weight.dtype)
    return out


HYPER = {"lr": 1e-3, "betas": (0.9, 0.95), "eps": 1e-8, "weight_decay": 0.1}


def _block_scale(blocks):
    """A power of two that brings the block's largest finite magnitude to [128, 256)."""
    largest = torch.where(blocks.isfinite(), blocks.abs(), 0.0).amax(1, keepdim=True)
    exponent = (largest.view(torch.int32) & 0x7F800000) - (7 << 23)  # in the bits of a 32-bit number
    return exponent.clamp(min=1 << 23).view(torch.float32)


def _first_8_bits(x):
    """The first moment: the nearest float8_e4m3fn of x over its block's scale."""
    blocks = x.view(-1, BLOCK)
    scale = _block_scale(blocks)
    return (blocks / scale).to(torch.float8_e4m3fn).view(-1), scale.view(-1)


def _hash(x):
    """32 bits of each (a multiply-xorshift mix), in 64-bit integers."""
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & 0xFFFFFFFF
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & 0xFFFFFFFF
    return x ^ (x >> 16)


def _key(seed, step):
    with_step = _hash(torch.tensor(seed & 0xFFFFFFFF)) ^ (step & 0xFFFFFFFF)
    return int(_hash(with_step))


def _uniform(n, seed, step):
    """One number of (0, 1) for each element, 16 bits each: two elements share the mix of their pair's index."""
    pair = _hash(torch.arange((n + 1) // 2, device=DEVICE) ^ _key(seed, step))
    return (torch.stack((pair & 0xFFFF, pair >> 16), 1).view(-1)[:n].float() + 0.5) * 2.0 ** -16


def _second_8_bits(x, u):
    """The second moment as its square root x: one of the two codes about x over the scale, chosen so that the square's
    mean is the second moment (its steps are far below a code's distance); a positive value keeps the smallest code."""
    blocks, u = x.view(-1, BLOCK), u.view(-1, BLOCK)
    scale = _block_scale(blocks)
    t = blocks / scale
    unit = (((t.view(torch.int32) & 0x7F800000).clamp(min=121 << 23)) - (3 << 23)).view(torch.float32)
    t = t / unit
    low = t.floor()
    code = (low + (t * t > low * low + u * (2 * low + 1))) * unit
    code = torch.where((code == 0.0) & (blocks > 0.0), 2.0 ** -9, code)
    return torch.where(blocks.isfinite(), code, float("nan")).to(torch.float8_e4m3fn).view(-1), scale.view(-1)


def _from_8_bits(q, scale):
    return (q.float().view(-1, BLOCK) * scale[:, None]).view(-1)


def _flat(tensors, spans, total):
    ends = [a for a, _ in spans[1:]] + [total]
    return torch.cat([torch.nn.functional.pad(t.reshape(-1).float(), (0, e - a - n))
                      for t, (a, n), e in zip(tensors, spans, ends)])


def _plain_adamw(s):
    case = s["case"]
    s["step"] += 1
    b1, b2 = HYPER["betas"]
    c1, c2 = 1 - b1 ** s["step"], 1 - b2 ** s["step"]
    p = s["master"] if case["master"] else _flat(s["params"], s["spans"], s["total"])
    g = _flat(s["grads"], s["spans"], s["total"])
    if case["bits"] == 8:
        m = _from_8_bits(s["exp_avg"], s["exp_avg_scale"])
        r = _from_8_bits(s["exp_avg_sq"], s["exp_avg_sq_scale"])
        v = r * r
    else:
        m, v = s["exp_avg"], s["exp_avg_sq"]
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * g) * (1 - b2)
    r = v.sqrt()
    p = p * (1 - HYPER["lr"] * HYPER["weight_decay"])
    p = p - m / (r * (1 / math.sqrt(c2)) + HYPER["eps"]) * (HYPER["lr"] / c1)
    if case["bits"] == 8:
        m, scale = _first_8_bits(m)
        s["exp_avg_scale"].copy_(scale)
        v, scale = _second_8_bits(r, _uniform(r.numel(), s["seed"], s["step"]))
        s["exp_avg_sq_scale"].copy_(scale)
    s["exp_avg"].copy_(m)
    s["exp_avg_sq"].copy_(v)
    if case["master"]:
        s["master"].copy_(p)
    torch._foreach_copy_(s["params"], [p[a:a + n].view(t.shape) for t, (a, n) in zip(s["params"], s["spans"])])


# ------------------------------------------------------------------------------------------------ one pass

def _own_logprobs(s):
    from mymyr_b200 import learn

    case = s["case"]
    got = learn.logprobs(s["logits"], s["tokens"], offsets=s.get("offsets"), mask=s.get("mask"),
                         temperature=case["temperature"], top=case["top"])
    out = {"logprob": got.logprob, "entropy": got.entropy}
    if case["top"]:
        out["top_logprobs"], out["top_tokens"] = got.top_logprobs, got.top_tokens
    if case["train"]:
        out["grad"], = torch.autograd.grad((got.logprob, got.entropy), s["logits"],
                                           (s["grad_logprob"], s["grad_entropy"]))
    return out


def _own_embedding(s):
    from mymyr_b200 import learn

    out = {"rows": learn.embedding(s["tokens"], s["weight"], scale=_scale(s["case"]))}
    if s["case"]["train"]:
        out["grad"], = torch.autograd.grad(out["rows"], s["weight"], s["grad"])
    return out


def _own_adamw(s):
    from mymyr_b200 import learn

    s["step"] += 1
    learn.adamw_step(s["params"], s["grads"], s["exp_avg"], s["exp_avg_sq"], step=s["step"], master=s.get("master"),
                     exp_avg_scale=s.get("exp_avg_scale"), exp_avg_sq_scale=s.get("exp_avg_sq_scale"),
                     seed=s["seed"], **HYPER)


def run(s):
    op = s["case"]["op"]
    if op == "adamw":
        if own:
            _own_adamw(s)
        else:
            with torch.no_grad():
                _plain_adamw(s)
        return {k: s[k] for k in ("params", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale", "master")
                if k in s}
    if own:
        return {"logprobs": _own_logprobs, "embedding": _own_embedding}[op](s)
    with torch.no_grad():
        return {"logprobs": _plain_logprobs, "embedding": _plain_embedding}[op](s)


# ------------------------------------------------------------------------------------------------ work

def work(case):
    """Each input read once, each output written once."""
    size = {"f32": 4, "bf16": 2, "f16": 2}[case["dtype"]]
    if case["op"] == "logprobs":
        rows = case["rows"]
        # ragged counts are squares of uniform ones: a third of the range on average
        count = rows * (case["least"] + (case["width"] - case["least"]) / 3) if case["ragged"] else rows * case["width"]
        io = count * size + rows * (8 + 4 + 4 + 12 * case["top"]) + (4 * rows if case["ragged"] else 0)
        io += count if case["masked"] else 0
        flops = 6 * count
        if case["train"]:
            io += count * size + 8 * rows
            flops += 6 * count
        return {"bytes": io, "flops": flops}
    if case["op"] == "embedding":
        n, v, w = case["tokens"], case["vocabulary"], case["width"]
        io = n * 8 + min(n, v) * w * size + n * w * size
        flops = n * w
        if case["train"]:
            io += n * w * size + v * w * size
            flops += n * w
        return {"bytes": io, "flops": flops}
    n = sum(math.prod(shape) for shape in _shapes(case))
    moments = 2 * 2 * (4 if case["bits"] == 32 else 1 + 4 / BLOCK)
    return {"bytes": n * (3 * size + moments + (8 - size if case["master"] else 0)), "flops": 16 * n}


# ------------------------------------------------------------------------------------------------ 64 bits

def _exact_logprobs(case, s):
    x, tokens, rows, top, t = s["logits"].detach(), s["tokens"], case["rows"], case["top"], case["temperature"]
    out = {"logprob": torch.zeros(rows, dtype=torch.float64, device=DEVICE),
           "entropy": torch.zeros(rows, dtype=torch.float64, device=DEVICE)}
    if top:
        out["top_tokens"] = None
        out["top_logprobs"] = torch.full((rows, top), -INF, dtype=torch.float64, device=DEVICE)
    if case["train"]:
        out["grad"] = torch.zeros(x.shape, dtype=torch.float64, device=DEVICE)
    width = case["width"]
    step = max(1, 2 ** 26 // width)
    for a in range(0, rows, step):
        b = min(rows, a + step)
        if case["ragged"]:
            lo, hi = s["offsets"][a:b].long()[:, None], s["offsets"][a + 1:b + 1].long()[:, None]
            at = lo + torch.arange(width, device=DEVICE)
            live = at < hi
            at = at.clamp(max=x.numel() - 1)
            z = x[at].double()
        else:
            live = s["mask"][a:b] if "mask" in s else torch.ones(b - a, width, dtype=torch.bool, device=DEVICE)
            z = x[a:b].double()
        z = torch.where(live, z / t, -INF)
        some = live.any(1)
        norm = torch.logsumexp(torch.where(some[:, None], z, 0.0), 1)
        lp = z - norm[:, None]
        lp[~some] = -INF
        q = lp.exp()
        h = torch.special.entr(q).sum(1)
        out["entropy"][a:b] = h
        y = tokens[a:b]
        one = torch.zeros_like(q)
        has = torch.nonzero(y >= 0)[:, 0]
        one[has, y[has]] = 1.0
        out["logprob"][a:b][has] = lp[has, y[has]]
        if top:
            k = min(top, width)
            out["top_logprobs"][a:b, :k] = lp.topk(k, dim=1).values
        if case["train"]:
            gl = s["grad_logprob"][a:b].double()[:, None] * (y >= 0)[:, None]
            ge = s["grad_entropy"][a:b].double()[:, None]
            z = gl * (one - q) - ge * q * (torch.where(live & some[:, None], lp, 0.0) + h[:, None])
            z = torch.where(live, z / t, 0.0)
            if case["ragged"]:
                out["grad"][at[live]] = z[live]
            else:
                out["grad"][a:b] = z
    return out


def _exact_embedding(case, s):
    tokens, w = s["tokens"], s["weight"].detach()
    has = torch.nonzero(tokens >= 0)[:, 0]
    out = {"rows": torch.zeros(tokens.numel(), w.shape[1], dtype=torch.float64, device=DEVICE)}
    out["rows"][has] = w[tokens[has]].double() * _scale(case)
    if case["train"]:
        out["grad"] = torch.zeros(w.shape, dtype=torch.float64, device=DEVICE)
        out["grad"].index_put_((tokens[has],), s["grad"][has].double() * _scale(case), accumulate=True)
    return out


def _mix(x):
    for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B)):
        x = ((x ^ (x >> shift)) * factor) % 2 ** 32
    return x ^ (x >> 16)


def _code(x, u=None):
    """Values of float8_e4m3fn for x over its block's scale, and the scales: the nearest one (ties to the even one), or
    for u the lower or the upper one by the squares' distances."""
    b = x.view(-1, BLOCK)
    top = b.abs().amax(1, keepdim=True)
    scale = torch.where(top > 0, 2.0 ** (top.log2().floor() - 7), 2.0 ** -126)
    b = b / scale
    unit = 2.0 ** ((torch.frexp(b).exponent - 1).clamp(min=-6) - 3).double()
    if u is None:
        return (torch.round(b / unit) * unit).view(-1), scale.view(-1)
    low = (b / unit).floor() * unit
    high = low + unit
    code = torch.where((b ** 2 - low ** 2) / (high ** 2 - low ** 2) > u.view(-1, BLOCK), high, low)
    code = torch.where((code == 0) & (b > 0), 2.0 ** -9, code)
    return code.view(-1), scale.view(-1)


def _exact_adamw(case, s):
    t = s["step"] + 1
    (b1, b2), lr, eps, decay = HYPER["betas"], HYPER["lr"], HYPER["eps"], HYPER["weight_decay"]
    n = s["total"]
    g, p = (torch.zeros(n, dtype=torch.float64, device=DEVICE) for _ in range(2))
    for i, (at, count) in enumerate(s["spans"]):
        g[at:at + count] = s["grads"][i].double().flatten()
        p[at:at + count] = s["params"][i].double().flatten()
    if case["master"]:
        p = s["master"].double()
    if case["bits"] == 8:
        m = (s["exp_avg"].double().view(-1, BLOCK) * s["exp_avg_scale"].double()[:, None]).flatten()
        v = (s["exp_avg_sq"].double().view(-1, BLOCK) * s["exp_avg_sq_scale"].double()[:, None]).flatten() ** 2
    else:
        m, v = s["exp_avg"].double(), s["exp_avg_sq"].double()
    m = b1 * m + (1 - b1) * g
    v = b2 * v + (1 - b2) * g * g
    update = (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + eps)
    p = p - lr * decay * p - lr * update
    out = {"params": [p[at:at + count].view(x.shape) for x, (at, count) in zip(s["params"], s["spans"])]}
    if case["bits"] == 8:
        key = _mix(_mix(s["seed"] % 2 ** 32) ^ t)
        at = torch.arange(n, device=DEVICE)
        u = _mix((at // 2) ^ key)
        u = torch.where(at % 2 == 0, u % 65536, u // 65536).double() / 65536 + 1 / 131072
        out["exp_avg"], out["exp_avg_scale"] = _code(m)
        out["exp_avg_sq"], out["exp_avg_sq_scale"] = _code(v.sqrt(), u)
    else:
        out["exp_avg"], out["exp_avg_sq"] = m, v
    if case["master"]:
        out["master"] = p
    return out


def exact(case, seed):
    s = prepare(case, seed)
    with torch.no_grad():
        return {"logprobs": _exact_logprobs, "embedding": _exact_embedding, "adamw": _exact_adamw}[case["op"]](case, s)
