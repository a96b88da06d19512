"""The learner's operators against plain computations in 64 bits: log-probabilities and their gradient, the embedding
lookup and its gradient, the AdamW step with moments in 32 and in 8 bits.

Tolerances come from the roundings a value goes through, EPS = 2^-24 each (32-bit arithmetic), plus half a unit in the
last place where the result is stored in 16 bits."""

import math

import numpy as np
import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from mymyr_b200 import _lib, learn, rl, tasks  # noqa: E402
from mymyr_b200.task import Task  # noqa: E402

INF = float("inf")
EPS = 2.0 ** -24
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HALF_ULP = {t: torch.finfo(t).eps / 2 for t in DTYPES}  # of the value: rounding to nearest
TINY = {t: torch.finfo(t).tiny * torch.finfo(t).eps / 2 for t in DTYPES}  # half the smallest subnormal number


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def randn(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=gen(seed), device="cuda") * scale


# ------------------------------------------------------------------------------------------------ log-probabilities

def plain(logits, tokens, mask, temperature, top, gl, ge):
    """Rows of logits [N, V] in 64 bits: log-probability, entropy, alternatives, the logits' gradient, and the spread of
    each row's finite logits (over T), which scales the rounding errors."""
    x = logits.double()
    x = torch.where(mask, x, -INF) if mask is not None else x
    n, width = x.shape
    best = x.amax(1, keepdim=True) if width else torch.full((n, 1), -INF, dtype=torch.float64, device="cuda")
    dead = best == -INF
    d = (x - torch.where(dead, 0.0, best)) / temperature
    s = d.exp().sum(1, keepdim=True)
    lp = torch.where(d == -INF, -INF, d - s.log())
    lp = torch.where(dead, -INF, lp)
    p = lp.exp()
    lp0 = torch.where(p > 0, lp, 0.0)
    h = -(p * lp0).sum(1)
    spread = torch.where(d == -INF, 0.0, -d).amax(1) if width else torch.zeros(n, dtype=torch.float64, device="cuda")
    given = tokens >= 0
    at = tokens.clamp(min=0, max=max(0, width - 1))
    rows = torch.arange(n, device="cuda")
    logp = torch.where(given, lp[rows, at] if width else torch.full((n,), -INF, device="cuda").double(), 0.0)
    order = torch.sort(x, dim=1, descending=True, stable=True)
    ids = torch.full((n, top), -1, dtype=torch.int64, device="cuda")
    values = torch.full((n, top), -INF, dtype=torch.float64, device="cuda")
    k = min(top, width)
    if k:
        live = order.values[:, :k] > -INF
        ids[:, :k] = torch.where(live, order.indices[:, :k], -1)
        values[:, :k] = torch.where(live, lp.gather(1, order.indices[:, :k]), -INF)
    g = torch.where(given, gl.double(), 0.0)[:, None]
    grad = -p * (g + ge.double()[:, None] * (lp0 + h[:, None]))
    if width:
        grad[rows, at] += torch.where(dead[:, 0], 0.0, g[:, 0])
    if mask is not None:
        grad = torch.where(mask, grad, 0.0)
    return logp, h, values, ids, torch.where(dead, 0.0, grad / temperature), p, spread


def near(got, want, tol):
    """Equal where not finite, within tol elsewhere."""
    got, want = got.double(), want.double()
    fin = want.float().isfinite()
    assert torch.equal(got.isfinite(), fin)
    assert torch.equal(got[~fin].nan_to_num(nan=5.0), want.float().double()[~fin].nan_to_num(nan=5.0))
    tol = tol.expand_as(want) if isinstance(tol, torch.Tensor) else torch.full_like(want, tol)
    over = (got - want).abs()[fin] - tol[fin]
    assert over.numel() == 0 or float(over.max()) <= 0, float(over.max())


def check_logprobs(logits, tokens, mask=None, temperature=1.0, top=0, seed=1):
    n = logits.shape[0]
    gl, ge = randn(n, seed=seed + 1), randn(n, seed=seed + 2, scale=0.5)
    want = plain(logits.detach(), tokens, mask, temperature, top, gl, ge)
    leaf = logits.detach().requires_grad_(True) if logits.is_contiguous() else logits.detach()
    leaf.requires_grad_(True)
    got = learn.logprobs(leaf, tokens, mask=mask, temperature=temperature, top=top)
    # (x - max) / T: three roundings of a number up to the spread (beyond 104 its exponential is zero); the sum of
    # exponentials: a chain below 64
    spread = want[6].clamp(max=104)
    tol = EPS * (4 * spread + 64)
    near(got.logprob, want[0], tol + 4 * EPS * want[0].abs().nan_to_num(posinf=0.0))
    near(got.entropy, want[1], tol * (2 + spread))
    if top:
        assert torch.equal(got.top_tokens, want[3])
        near(got.top_logprobs, want[2], tol[:, None] + 4 * EPS * want[2].abs().nan_to_num(posinf=0.0))
    grad, = torch.autograd.grad((got.logprob, got.entropy), leaf, (gl, ge))
    size = (gl.abs()[:, None] + ge.abs()[:, None] * (spread + want[1] + 1)[:, None]) / temperature
    bound = tol[:, None] * 4 * size * want[5] + HALF_ULP[leaf.dtype] * want[4].abs() * 1.01 + 2 * TINY[leaf.dtype]
    bound = bound + 4 * EPS * size * (want[5] + (want[4] != 0))  # the token's own 1 - p
    near(grad, want[4], bound)
    none = learn.logprobs(leaf.detach(), tokens, mask=mask, temperature=temperature, top=top)
    assert torch.equal(none.logprob.nan_to_num(), got.logprob.nan_to_num())
    assert torch.equal(none.entropy.nan_to_num(), got.entropy.nan_to_num())


def some_tokens(n, width, seed):
    t = torch.randint(0, width, (n,), generator=gen(seed), device="cuda")
    if n > 2:
        t[n // 2] = -1
    return t


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("width", [1, 2, 3, 7, 8, 31, 33, 64, 255, 257, 1000, 1023, 2048, 4099])
@pytest.mark.parametrize("rows,top", [(1, 5), (5, 0), (67, 32)])
def test_logprobs_dense(dtype, width, rows, top):
    x = randn(rows, width, seed=width, scale=3.0).to(dtype)
    check_logprobs(x, some_tokens(rows, width, 3), temperature=0.7 if width % 2 else 1.0, top=top)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(1, 40001), (1, 131072), (2, 65537), (3, 32768), (9, 50000), (40, 30001),
                                        (300, 9001), (600, 5000)])
def test_logprobs_wide(dtype, rows, width):
    x = randn(rows, width, seed=width, scale=2.0).to(dtype)
    check_logprobs(x, some_tokens(rows, width, 3), temperature=1.3, top=20)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(4, 1), (9, 40), (33, 1001), (6, 16384), (2, 70003)])
def test_logprobs_masked(dtype, rows, width):
    x = randn(rows, width, seed=width, scale=2.0).to(dtype)
    mask = torch.rand(rows, width, generator=gen(5), device="cuda") < 0.4
    mask[0] = False           # nothing left
    mask[1] = False
    mask[1, width // 2] = True  # one left
    x[~mask] = torch.tensor([float("nan"), INF, -INF, 1e4], device="cuda", dtype=dtype)[
        torch.arange(int((~mask).sum()), device="cuda") % 4]  # what lies under the mask does not count
    check_logprobs(x, some_tokens(rows, width, 3), mask=mask, top=8)


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("rows,width", [(5, 9), (3, 1200), (4, 33000)])
def test_logprobs_lowest_values_and_infinities(dtype, rows, width):
    low = torch.finfo(dtype).min
    x = randn(rows, width, seed=2).to(dtype)
    x[:, ::2] = -INF          # a mask by infinities
    x[1] = -INF               # a row of them: nothing left
    x[2], x[2, 0] = low, 1.0  # a mask by the type's lowest value
    x[0] = low                # a row of it: even odds
    for t in (1.0, 0.5):
        check_logprobs(x, some_tokens(rows, width, 3), temperature=t, top=3)


@pytest.mark.parametrize("rows,width", [(3, 12), (2, 3000), (1, 50000)])
def test_logprobs_nan_and_plus_infinity_spoil_their_row_alone(rows, width):
    for bad in (float("nan"), INF):
        x = randn(rows + 2, width, seed=1)
        x[1, width // 3] = bad
        y = torch.zeros(rows + 2, dtype=torch.int64, device="cuda")
        clean = learn.logprobs(x[2:].contiguous(), y[2:], top=4)
        leaf = x.requires_grad_(True)
        got = learn.logprobs(leaf, y, top=4)
        g, = torch.autograd.grad(got.logprob.sum(), leaf)
        assert got.logprob[1].isnan() and got.entropy[1].isnan() and got.top_logprobs[1].isnan().all()
        assert (got.top_tokens[1] == -1).all() and g[1].isnan().all()
        assert torch.equal(got.logprob[2:], clean.logprob) and torch.equal(got.top_tokens[2:], clean.top_tokens)
        assert g[0].isfinite().all() and g[2:].isfinite().all()


@pytest.mark.parametrize("width", [5, 40, 700, 5000, 100000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_logprobs_ties_go_to_the_lowest_index(width, dtype):
    x = torch.zeros(3, width, dtype=dtype, device="cuda")
    x[1] = (torch.arange(width, device="cuda") % 3).to(dtype)
    x[2] = randn(width, seed=1).round().to(dtype)
    x[2, ::7] = -0.0
    got = learn.logprobs(x, torch.zeros(3, dtype=torch.int64, device="cuda"), top=32)
    want = torch.sort(x.float(), dim=1, descending=True, stable=True).indices[:, :32]
    k = min(32, width)
    assert torch.equal(got.top_tokens[:, :k], want[:, :k])
    assert (got.top_tokens[:, k:] == -1).all() and (got.top_logprobs[:, k:] == -INF).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_logprobs_sorted_rows_keep_every_alternative(dtype):
    """The best ones all in one place of the row, at its start, its end and in its middle."""
    width = 20000
    x = randn(4, width, seed=1).to(dtype)
    x[0, :40] = torch.linspace(9, 8, 40, device="cuda").to(dtype)
    x[1, -40:] = torch.linspace(8, 9, 40, device="cuda").to(dtype)
    x[2, 9000:9040] = 9.0
    x[3] = torch.linspace(-8, 8, width, device="cuda").to(dtype)
    check_logprobs(x, some_tokens(4, width, 3), top=32)


def test_logprobs_strides_offsets_and_shapes():
    base = randn(40, 300, seed=1)
    y = some_tokens(40, 64, 2)
    for view in (base[:, 1:65], base[:, 3:67], base[:, :128:2], randn(64, 40, seed=3).t(), base[:1, :64].expand(40, 64),
                 base.bfloat16()[:, 5:69], base.half()[:, 1:65]):
        check_logprobs(view, y, top=4)
    # a mask of one row for all, of the logits' rows, of strided rows
    x = randn(40, 64, seed=4)
    one = torch.rand(64, generator=gen(1), device="cuda") < 0.5
    got = learn.logprobs(x, y, mask=one, top=3)
    want = learn.logprobs(x, y, mask=one.expand(40, 64).contiguous(), top=3)
    wide = torch.zeros(40, 131, dtype=torch.bool, device="cuda")
    wide[:, 3:67] = one
    strided = learn.logprobs(x, y, mask=wide[:, 3:67], top=3)
    for other in (want, strided):
        assert torch.equal(got.logprob, other.logprob) and torch.equal(got.top_tokens, other.top_tokens)
        assert torch.equal(got.entropy, other.entropy)
    # leading dimensions, tokens of 32 bits, no tokens
    z = learn.logprobs(x.view(5, 8, 64), y.view(5, 8).int(), top=2)
    flat = learn.logprobs(x, y, top=2)
    assert z.logprob.shape == (5, 8) and z.top_tokens.shape == (5, 8, 2)
    assert torch.equal(z.logprob.view(-1), flat.logprob) and torch.equal(z.top_tokens.view(40, 2), flat.top_tokens)
    single = learn.logprobs(x[7], y[7])
    assert single.logprob.shape == () and torch.equal(single.logprob, flat.logprob[7])
    assert learn.logprobs(x).logprob is None
    assert torch.equal(learn.logprobs(x).entropy, flat.entropy)


def test_logprobs_empty_inputs_and_tokens_past_the_row():
    for n, v in ((0, 7), (3, 0)):
        x = torch.zeros(n, v, device="cuda", requires_grad=True)
        got = learn.logprobs(x, torch.full((n,), -1, device="cuda"), top=2)
        assert got.logprob.shape == (n,) and (got.entropy == 0).all() and (got.top_tokens == -1).all()
        g, = torch.autograd.grad(got.entropy.sum(), x)
        assert g.shape == x.shape
    x = randn(3, 10, seed=1).requires_grad_(True)
    y = torch.tensor([2, 10, -7], device="cuda")
    got = learn.logprobs(x, y)
    assert got.logprob[0].isfinite() and got.logprob[1].isnan() and got.logprob[2] == 0
    g, = torch.autograd.grad(got.logprob.sum(), x)
    assert g[0].isfinite().all() and g[1].isnan().all() and (g[2] == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", [[0], [1], [3, 0, 2, 2, 4] * 50, [0, 0, 5000, 1, 17], [40] * 9, [300, 0, 1100, 700],
                                    [2, 3] * 700, [30000, 1, 0, 12345]])
def test_logprobs_ragged(dtype, counts):
    offsets = torch.tensor([0] + list(np.cumsum(counts)), dtype=torch.int32, device="cuda")
    n, total, width = len(counts), int(sum(counts)), max(counts)
    flat = randn(max(total, 1), seed=total, scale=2.0)[:total].to(dtype)
    tokens = torch.tensor([c - 1 if c else -1 for c in counts], dtype=torch.int64, device="cuda")
    gl, ge = randn(n, seed=1), randn(n, seed=2)
    # the same rows, padded by minus infinity
    x = torch.full((n, max(width, 1)), -INF, dtype=torch.float64, device="cuda")
    at = 0
    for i, c in enumerate(counts):
        x[i, :c] = flat[at:at + c].double()
        at += c
    want = plain(x, tokens, None, 1.0, 6, gl, ge)
    for off in (offsets, offsets.long()):
        leaf = flat.clone().requires_grad_(True)
        got = learn.logprobs(leaf, tokens, offsets=off, top=6)
        tol = EPS * (4 * want[6] + 64)
        near(got.logprob, want[0], tol)
        near(got.entropy, want[1], tol * (2 + want[6]))
        assert torch.equal(got.top_tokens, want[3])
        near(got.top_logprobs, want[2], tol[:, None])
        grad, = torch.autograd.grad((got.logprob, got.entropy), leaf, (gl, ge))
        at = 0
        for i, c in enumerate(counts[:20]):
            w, p = want[4][i, :c], want[5][i, :c]
            size = gl[i].abs() + ge[i].abs() * (want[6][i] + want[1][i] + 1)
            bound = tol[i] * 4 * size * p + HALF_ULP[dtype] * w.abs() * 1.01 + 2 * TINY[dtype]
            near(grad[at:at + c], w, bound + 4 * EPS * size * (p + (w != 0)))
            at += c


def test_logprobs_ragged_masked_and_untrue_offsets():
    counts = [5, 0, 40, 3]
    offsets = torch.tensor([0, 5, 5, 45, 48], device="cuda")
    flat = randn(60, seed=1)  # the last twelve belong to no row
    mask = torch.rand(60, generator=gen(2), device="cuda") < 0.5
    y = torch.tensor([0, -1, 3, 1], device="cuda")
    leaf = flat.clone().requires_grad_(True)
    got = learn.logprobs(leaf, y, offsets=offsets, mask=mask, top=3)
    low = learn.logprobs(flat.masked_fill(~mask, -INF), y, offsets=offsets, top=3)
    assert torch.equal(got.logprob, low.logprob) and torch.equal(got.top_tokens, low.top_tokens)
    g, = torch.autograd.grad(got.entropy.sum(), leaf)
    assert (g[48:] == 0).all() and (g[~mask] == 0).all()
    # offsets that run backwards or past the vector are cut to it
    wild = torch.tensor([-4, 9, 3, 4000, 2 ** 40], device="cuda")
    cut = torch.tensor([[0, 9], [9, 9], [3, 60], [60, 60]])
    got = learn.logprobs(flat, offsets=wild, top=1)
    for i, (b, e) in enumerate(cut.tolist()):
        want = learn.logprobs(flat[b:e][None], top=1)
        assert torch.allclose(got.entropy[i], want.entropy[0], atol=1e-5)
        assert int(got.top_tokens[i, 0]) == int(want.top_tokens[0, 0])


@pytest.mark.parametrize("rows,width", [(6, 5), (4, 300), (2, 9000)])
def test_logprobs_gradient_against_differences(rows, width):
    """Along a direction of unit length, h = 2^-5: the sums' own errors (2^-18 for each row) over 2 h stay below 2^-13
    for each row, the third derivative's part below h^2."""
    x = randn(rows, width, seed=1)
    y = some_tokens(rows, width, 2)
    gl, ge = randn(rows, seed=3), randn(rows, seed=4)
    way = randn(rows, width, seed=5)
    way = way / way.norm(dim=1, keepdim=True)

    def loss(z):
        got = learn.logprobs(z, y, temperature=0.8)
        return (got.logprob.double() * gl + got.entropy.double() * ge).sum()

    leaf = x.clone().requires_grad_(True)
    grad, = torch.autograd.grad(loss(leaf), leaf)
    h = 2.0 ** -5
    diff = float((loss(x + h * way) - loss(x - h * way)) / (2 * h))
    assert abs(diff - float((grad.double() * way).sum())) <= rows * (2.0 ** -13 + h * h)


def test_logprobs_gradients_of_one_output_and_of_broadcast_ones():
    x = randn(7, 90, seed=1)
    y = some_tokens(7, 90, 2)
    full = []
    for pick in ("logprob", "entropy"):
        leaf = x.clone().requires_grad_(True)
        g, = torch.autograd.grad(getattr(learn.logprobs(leaf, y), pick).sum(), leaf)  # an expanded gradient of ones
        full.append(g)
    leaf = x.clone().requires_grad_(True)
    got = learn.logprobs(leaf, y)
    both, = torch.autograd.grad(got.logprob.sum() + got.entropy.sum(), leaf)
    assert torch.allclose(both, full[0] + full[1], atol=1e-6)
    row = x[:1].clone().requires_grad_(True)  # one row for all: its gradient is the sum
    g, = torch.autograd.grad(learn.logprobs(row.expand(7, 90), y).logprob.sum(), row)
    leaf = x[:1].expand(7, 90).clone().requires_grad_(True)
    each, = torch.autograd.grad(learn.logprobs(leaf, y).logprob.sum(), leaf)
    assert torch.allclose(g, each.sum(0, keepdim=True), atol=1e-5)


def test_logprobs_past_32_bit_offsets():
    """A row whose logits lie past 2^32 elements (half a row of them in front), bf16: 8.6 GB."""
    free, _ = torch.cuda.mem_get_info()
    if free < 12 << 30:
        pytest.skip("needs 12 GB")
    big = torch.zeros(2, 2 ** 31 + 8, dtype=torch.bfloat16, device="cuda")
    width = 1000
    view = big[:, -width:]
    view.copy_(randn(2, width, seed=1))
    y = some_tokens(2, width, 2)
    got = learn.logprobs(view, y, top=3)
    want = learn.logprobs(view.contiguous(), y, top=3)
    assert torch.equal(got.logprob, want.logprob) and torch.equal(got.top_tokens, want.top_tokens)


# ------------------------------------------------------------------------------------------------ embeddings

@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("n,vocabulary,width", [(1, 1, 1), (1, 5, 8), (7, 3, 5), (64, 1000, 64), (300, 7, 33),
                                                (1000, 300, 128), (4097, 70000, 16), (5000, 2, 24), (9000, 513, 1000),
                                                (33, 2 ** 17, 2048), (20000, 40, 2), (70000, 9, 17)])
def test_embedding(dtype, n, vocabulary, width):
    w = randn(vocabulary, width, seed=n).to(dtype)
    tokens = torch.randint(0, vocabulary, (n,), generator=gen(n), device="cuda")
    if n > 3:
        tokens[:: max(2, n // 9)] = -1
        tokens[n // 2:n // 2 + n // 4] = vocabulary - 1  # a long run of one token
    g = randn(n, width, seed=n + 1).to(dtype)
    leaf = w.clone().requires_grad_(True)
    got = learn.embedding(tokens, leaf, scale=1.5)
    held = (tokens >= 0)[:, None]
    want = torch.where(held, (w[tokens.clamp(min=0)].float() * 1.5), 0.0).to(dtype)  # one rounding: the same bits
    assert torch.equal(got, want)
    grad, = torch.autograd.grad(got, leaf, g)
    at = tokens[held[:, 0]]
    total = torch.zeros(vocabulary, width, dtype=torch.float64, device="cuda")
    size = torch.zeros_like(total)
    total.index_put_((at,), g[held[:, 0]].double() * 1.5, accumulate=True)
    size.index_put_((at,), g[held[:, 0]].double().abs() * 1.5, accumulate=True)
    most = int(torch.bincount(at, minlength=1).max()) if at.numel() else 1
    # a sum of `most` terms: at most that many roundings, of sums no larger than the sum of magnitudes
    tol = size * EPS * (most + 2) + HALF_ULP[dtype] * total.abs() * 1.01 + 2 * TINY[dtype]
    near(grad, total, tol)
    again, = torch.autograd.grad(learn.embedding(tokens.int(), leaf, scale=1.5), leaf, g)
    assert torch.equal(grad, again)  # in the same order on every call, whatever the tokens' type


@pytest.mark.parametrize("n", [200000, 300001])
@pytest.mark.parametrize("vocabulary", [1, 3, 20000, 2 ** 20])
def test_embedding_gradient_of_many_tokens(n, vocabulary):
    width = 4
    tokens = (torch.rand(n, generator=gen(1), device="cuda") ** 4 * vocabulary).long().clamp(max=vocabulary - 1)
    g = torch.randint(-4, 5, (n, width), generator=gen(2), device="cuda").float()  # whole numbers: exact sums
    w = torch.zeros(vocabulary, width, device="cuda", requires_grad=True)
    grad, = torch.autograd.grad(learn.embedding(tokens, w), w, g)
    want = torch.zeros(vocabulary, width, dtype=torch.float64, device="cuda")
    want.index_put_((tokens,), g.double(), accumulate=True)
    assert torch.equal(grad.double(), want)


def test_embedding_strides_shapes_and_tokens_outside():
    table = randn(50, 100, seed=1)
    tokens = torch.tensor([[0, 49, -1], [50, 2 ** 40, -2 ** 40]], device="cuda")
    got = learn.embedding(tokens, table[:, 3:20])
    assert got.shape == (2, 3, 17)
    assert torch.equal(got[0, :2], table[[0, 49], 3:20]) and (got[0, 2] == 0).all() and (got[1, 2] == 0).all()
    assert got[1, :2].isnan().all()
    turned = randn(17, 50, seed=2).t()
    assert torch.equal(learn.embedding(tokens[0, :2], turned), turned[[0, 49]])
    w = table.clone().requires_grad_(True)
    g, = torch.autograd.grad(learn.embedding(tokens, w, scale=2.0).nan_to_num().sum(), w)  # an expanded gradient
    assert (g[0] == 2).all() and (g[49] == 2).all() and (g[1:49] == 0).all()
    rows = learn.embedding(tokens[0], w)
    odd = randn(3, 250, seed=3)[:, 1:201:2]  # columns two apart
    g, = torch.autograd.grad(rows, w, odd)
    assert torch.equal(g[0], odd[0]) and torch.equal(g[49], odd[1])
    for shape in ((0,), (2, 0)):
        none = learn.embedding(torch.zeros(shape, dtype=torch.int64, device="cuda"), w)
        assert none.shape == (*shape, 100)
        g, = torch.autograd.grad(none.sum(), w)
        assert (g == 0).all()
    assert learn.embedding(torch.tensor(3, device="cuda"), table).shape == (100,)


def test_embedding_gradient_against_differences():
    """The loss is linear in the table: one difference gives the derivative up to its sums' roundings."""
    w, tokens = randn(30, 12, seed=1), torch.randint(-1, 30, (200,), generator=gen(2), device="cuda")
    g, way = randn(200, 12, seed=3), randn(30, 12, seed=4)
    leaf = w.clone().requires_grad_(True)
    grad, = torch.autograd.grad(learn.embedding(tokens, leaf, scale=0.5), leaf, g)
    up, down = (learn.embedding(tokens, w + s * way, scale=0.5).double() for s in (1.0, -1.0))
    diff = float(((up - down) / 2 * g).sum())
    size = float((up.abs() + down.abs()).mul(g.abs()).sum())
    assert abs(diff - float((grad.double() * way).sum())) <= 8 * EPS * size


def test_embedding_past_32_bit_offsets():
    """A table of 4.6 G elements, bf16: 9.2 GB, and its gradient."""
    free, _ = torch.cuda.mem_get_info()
    if free < 24 << 30:
        pytest.skip("needs 24 GB")
    vocabulary, width = 70000, 65536
    w = torch.zeros(vocabulary, width, dtype=torch.bfloat16, device="cuda")
    tokens = torch.tensor([69999, 5, 69999], device="cuda")
    w[69999] = randn(width, seed=1)
    w.requires_grad_(True)
    rows = learn.embedding(tokens, w)
    assert torch.equal(rows[0], w[69999]) and torch.equal(rows[2], w[69999]) and (rows[1] == 0).all()
    g = torch.ones_like(rows)
    grad, = torch.autograd.grad(rows, w, g)
    assert (grad[69999] == 2).all() and (grad[5] == 1).all() and float(grad.sum(dtype=torch.float64)) == 3 * width


# ------------------------------------------------------------------------------------------------ AdamW

SHAPES = [(1,), (255,), (256,), (257,), (3, 5), (40, 33), (0,), (1000, 7), (4096,), (70001,)]


def moments_of(state, name):
    x = state[name].double()
    return x if state[name].dtype == torch.float32 else \
        (x.view(-1, learn.BLOCK) * state[name + "_scale"].double()[:, None]).view(-1)


def flat_of(tensors, total):
    out, at = torch.zeros(total, dtype=torch.float64, device="cuda"), 0
    for t in tensors:
        out[at:at + t.numel()] = t.detach().double().reshape(-1)
        at += -(-t.numel() // learn.BLOCK) * learn.BLOCK
    return out


def pow2(e):
    """2 to a 64-bit tensor of exponents, exactly."""
    return ((e.long() + 1023) << 52).view(torch.float64)


def mix(x):
    for shift, factor in ((16, 0x7FEB352D), (15, 0x846CA68B)):
        x = ((x ^ (x >> shift)) * factor) & 0xFFFFFFFF
    return x ^ (x >> 16)


def uniforms(n, seed, step):
    key = mix(mix(seed) ^ step)
    at = np.arange(n, dtype=np.int64)
    h = mix((at >> 1) ^ key)
    return torch.from_numpy((np.where(at % 2 == 0, h & 0xFFFF, h >> 16) + 0.5) / 65536).cuda()


@pytest.mark.parametrize("dtype,grad_dtype,master", [(torch.float32, torch.float32, False),
                                                     (torch.bfloat16, torch.bfloat16, False),
                                                     (torch.float16, torch.float16, True),
                                                     (torch.bfloat16, torch.float32, True),
                                                     (torch.float16, torch.float32, False)])
@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_step(dtype, grad_dtype, master, bits):
    shapes = SHAPES * 3
    params = [randn(*s, seed=i).to(dtype) for i, s in enumerate(shapes)]
    state = learn.adamw_state(params, bits=bits, master=master)
    total = state["exp_avg"].numel()
    hyper = dict(lr=3e-3, betas=(0.9, 0.97), eps=1e-6, weight_decay=0.1)
    for step in range(1, 5):
        grads = [(randn(*s, seed=100 * step + i) * 10.0 ** -(i % 5)).to(grad_dtype) for i, s in enumerate(shapes)]
        g = flat_of(grads, total)
        p = state["master"].double() if master else flat_of(params, total)
        m, r = moments_of(state, "exp_avg"), moments_of(state, "exp_avg_sq")
        v = r * r if bits == 8 else r
        learn.adamw_step(params, grads, step=step, seed=9, **hyper, **state)
        b1, b2 = hyper["betas"]
        # three roundings of each part; the betas are themselves rounded to 32 bits
        m_size = (m * b1).abs() + (g * (1 - b1)).abs()
        m, v = m * b1 + g * (1 - b1), v * b2 + g * g * (1 - b2)
        new = p * (1 - hyper["lr"] * 0.1)
        move = m / (1 - b1 ** step) / ((v / (1 - b2 ** step)).sqrt() + hyper["eps"]) * hyper["lr"]
        part = m_size / (1 - b1 ** step) / ((v / (1 - b2 ** step)).sqrt() + hyper["eps"]) * hyper["lr"]
        tol = 4 * EPS * p.abs() + 24 * EPS * part
        if master:
            near(state["master"], new - move, tol)
        now = flat_of(params, total)
        near(now, new - move, tol + (0 if dtype == torch.float32 else
                                     HALF_ULP[dtype] * (new - move).abs() * 1.01 + 2 * TINY[dtype]))
        if bits == 32:
            near(state["exp_avg"], m, 6 * EPS * m_size)
            near(state["exp_avg_sq"], v, 8 * EPS * v)
            continue
        r = v.sqrt()
        u = uniforms(total, 9, step)
        for name, x in (("exp_avg", m), ("exp_avg_sq", r)):
            scale = state[name + "_scale"].double()
            top = x.view(-1, learn.BLOCK).abs().amax(1)
            assert (torch.frexp(scale).mantissa == 0.5).all()
            held = top > 0
            ratio = top[held] / scale[held]
            assert float(ratio.min()) >= 128 * (1 - 8 * EPS) and float(ratio.max()) < 256 * (1 + 8 * EPS)
            x = (x.view(-1, learn.BLOCK) / scale[:, None]).view(-1)
            code = state[name].double()
            unit = pow2((torch.frexp(x).exponent - 1).clamp(min=-6) - 3)
            if name == "exp_avg":
                rounded = m_size / scale.repeat_interleave(learn.BLOCK) * 6 * EPS
                near(code, x, unit / 2 + rounded)
                continue
            low = (x / unit).floor() * unit
            want = torch.where((x * x - low * low) / ((low + unit) ** 2 - low * low) > u, low + unit, low)
            want = torch.where((want == 0) & (x > 0), 2.0 ** -9, want)
            # a few values lie so near a boundary that 32 bits may take the other side: 2^-18 of the distance
            edge = ((x * x - low * low) / ((low + unit) ** 2 - low * low) - u).abs() < 2.0 ** -14
            edge |= (x / unit - (x / unit).round()).abs() < 2.0 ** -14
            edge &= x > 0
            assert torch.equal(code[~edge], want[~edge]) and float(edge.double().mean()) < 1e-2
            near(code[edge], x[edge], unit[edge] * 1.01 + 2.0 ** -9)


def test_adamw_rounds_the_second_moment_without_bias():
    """4,096 blocks, one element sets each scale; the squares of the others' codes average to the second moment within
    five standard deviations (at most half the distance of two squares, over the square root of their number)."""
    n = 4096 * 256
    p, g = torch.zeros(n, device="cuda"), torch.full((n,), 0.37, device="cuda")
    g[::256] = 5.0
    state = learn.adamw_state([p], bits=8)
    learn.adamw_step([p], [g], step=1, betas=(0.9, 0.99), lr=0.0, seed=4, **state)
    r = moments_of(state, "exp_avg_sq").view(-1, 256)[:, 1:]
    want = 0.01 * 0.37 ** 2
    low, high = float(r.min()), float(r.max())
    assert low < math.sqrt(want) < high and (high - low) / low < 0.13
    assert abs(float((r * r).mean()) - want) < 5 * (high ** 2 - low ** 2) / 2 / math.sqrt(r.numel())
    again = learn.adamw_state([p], bits=8)
    learn.adamw_step([p], [g], step=1, betas=(0.9, 0.99), lr=0.0, seed=5, **again)
    assert not torch.equal(again["exp_avg_sq"].float(), state["exp_avg_sq"].float())  # another seed


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_skips_missing_gradients_and_keeps_bad_ones_to_themselves(bits):
    params = [randn(700, seed=1), randn(300, seed=2), randn(5, seed=3)]
    before = [p.clone() for p in params]
    state = learn.adamw_state(params, bits=bits)
    g = randn(700, seed=4)
    g[3], g[600] = float("nan"), INF
    learn.adamw_step(params, [g, None, torch.zeros(5, device="cuda")], step=1, weight_decay=0.0, **state)
    assert torch.equal(params[1], before[1]) and torch.equal(params[2], before[2])
    bad = torch.zeros(700, dtype=torch.bool, device="cuda")
    bad[3] = bad[600] = True
    assert params[0][~bad].isfinite().all() and not params[0][bad].isfinite().any()
    m = moments_of(state, "exp_avg")
    assert m[:700][~bad].isfinite().all() and not m[:700][bad].isfinite().any() and (m[700:] == 0).all()


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_alignment_and_many_tensors(bits):
    """Tensors at odd places of one array, and more of them than one launch takes: as each alone would be."""
    store, grads = randn(9000, seed=1), randn(9000, seed=2)
    cuts = [(1, 900), (901, 4000), (4003, 4004), (4100, 9000)]
    params = [store[a:b] for a, b in cuts]
    apart = [p.clone() for p in params]
    state, other = learn.adamw_state(params, bits=bits), learn.adamw_state(apart, bits=bits)
    for step in (1, 2):
        learn.adamw_step(params, [grads[a:b] for a, b in cuts], step=step, **state)
        learn.adamw_step(apart, [grads[a:b].clone() for a, b in cuts], step=step, **other)
    for a, b in zip(params, apart):
        assert torch.equal(a, b)
    for k in state:
        assert torch.equal(state[k].float(), other[k].float())
    assert torch.equal(store[4004:4100], randn(9000, seed=1)[4004:4100])
    many = [randn(1 + i % 300, seed=i) for i in range(2100)]
    gs = [randn(1 + i % 300, seed=i + 7) for i in range(2100)]
    few = [p.clone() for p in many]
    state = learn.adamw_state(many, bits=bits)
    learn.adamw_step(many, gs, step=3, **state)
    for i in (0, 95, 96, 999, 1000, 1001, 2000, 2099):
        learn.adamw_step([few[i]], [gs[i]], step=3, **learn.adamw_state([few[i]], bits=bits))
        assert torch.equal(few[i], many[i])


def test_adamw_object_groups_and_state():
    def make():
        a, b = randn(30, 20, seed=1).requires_grad_(True), randn(20, seed=2).requires_grad_(True)
        return a, b, learn.AdamW([{"params": [a]}, {"params": [b], "weight_decay": 0.0, "lr": 1e-2}], lr=1e-3,
                                 weight_decay=0.5)

    a, b, opt = make()
    ra, rb = a.detach().clone().requires_grad_(True), b.detach().clone().requires_grad_(True)
    ref = torch.optim.AdamW([{"params": [ra], "weight_decay": 0.5}, {"params": [rb], "weight_decay": 0.0, "lr": 1e-2}],
                            lr=1e-3)
    x = randn(8, 30, seed=3, scale=0.1)
    for i in range(6):
        for p, q, o in ((a, b, opt), (ra, rb, ref)):
            o.zero_grad()
            ((x @ p + q).tanh() ** 2).sum().backward()
            o.step()
        if i == 2:
            saved = {k: v for k, v in opt.state_dict().items()}
            saved["state"] = [{k: t.clone() for k, t in s.items()} for s in saved["state"]]
            at = a.detach().clone(), b.detach().clone()
    assert torch.allclose(a, ra, atol=2e-6) and torch.allclose(b, rb, atol=2e-6)
    a2, b2, opt2 = make()
    with torch.no_grad():
        a2.copy_(at[0])
        b2.copy_(at[1])
    opt2.load_state_dict(saved)
    for _ in range(3):
        opt2.zero_grad()
        ((x @ a2 + b2).tanh() ** 2).sum().backward()
        opt2.step()
    assert torch.equal(a, a2) and torch.equal(b, b2)


# ------------------------------------------------------------------------------------------------ use

def test_streams_and_graphs():
    """On another stream than torch's current one, and captured in a CUDA graph: the same bits."""
    x, y = randn(50, 3000, seed=1), some_tokens(50, 3000, 2)
    w, t = randn(500, 64, seed=3), torch.randint(0, 500, (999,), generator=gen(4), device="cuda")
    want = learn.logprobs(x, y, top=4)
    rows = learn.embedding(t, w)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    got = learn.logprobs(x, y, top=4, stream=s.cuda_stream)
    other = learn.embedding(t, w, stream=s.cuda_stream)
    s.synchronize()
    assert torch.equal(got.logprob, want.logprob) and torch.equal(got.top_tokens, want.top_tokens)
    assert torch.equal(other, rows)

    leaf, table, g = x.clone().requires_grad_(True), w.clone().requires_grad_(True), randn(999, 64, seed=5)

    def step():
        out = learn.logprobs(leaf, y)
        gx, = torch.autograd.grad((out.logprob, out.entropy), leaf, (ones, ones))
        gw, = torch.autograd.grad(learn.embedding(t, table), table, g)
        return gx, gw

    ones = torch.ones(50, device="cuda")
    plain_gx, plain_gw = step()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        gx, gw = step()
    gx.zero_()
    gw.fill_(7.0)
    for _ in range(2):
        graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(gx, plain_gx) and torch.equal(gw, plain_gw)


def test_refusals():
    x, y = randn(4, 8, seed=1), torch.zeros(4, dtype=torch.int64, device="cuda")
    off = torch.zeros(5, dtype=torch.int64, device="cuda")
    for bad in (lambda: learn.logprobs(x.double(), y), lambda: learn.logprobs(x.cpu(), y),
                lambda: learn.logprobs(x, y.float()), lambda: learn.logprobs(x, y[:3]),
                lambda: learn.logprobs(x, y.cpu()), lambda: learn.logprobs(x, y, temperature=0.0),
                lambda: learn.logprobs(x, y, temperature=-1.0), lambda: learn.logprobs(x, y, temperature=INF),
                lambda: learn.logprobs(x, y, temperature=float("nan")), lambda: learn.logprobs(x, y, top=33),
                lambda: learn.logprobs(x, y, top=-1), lambda: learn.logprobs(x, y, mask=x),
                lambda: learn.logprobs(x, y, offsets=off), lambda: learn.logprobs(x[0], y, offsets=off.float()),
                lambda: learn.logprobs(x, y, mask=torch.ones(2, 4, 8, dtype=torch.bool, device="cuda")),
                lambda: learn.logprobs(torch.tensor(1.0, device="cuda")),
                lambda: learn.embedding(y.float(), x), lambda: learn.embedding(y, x[0]),
                lambda: learn.embedding(y, x.long()), lambda: learn.embedding(y.cpu(), x),
                lambda: learn.adamw_state([]), lambda: learn.adamw_state([x], bits=4),
                lambda: learn.adamw_state([x.long()])):
        with pytest.raises((ValueError, RuntimeError)):
            bad()
    state = learn.adamw_state([x])
    eight = learn.adamw_state([x], bits=8)
    for bad in (lambda: learn.adamw_step([x], [], step=1, **state), lambda: learn.adamw_step([x], [x], step=0, **state),
                lambda: learn.adamw_step([x], [x[:2]], step=1, **state),
                lambda: learn.adamw_step([x.t()], [x.t()], step=1, **state),
                lambda: learn.adamw_step([x], [x.half()], step=1, **state),
                lambda: learn.adamw_step([x, x.clone()], [x, x], step=1, **state),
                lambda: learn.adamw_step([x], [x], state["exp_avg"], state["exp_avg_sq"][:8], step=1),
                lambda: learn.adamw_step([x], [x], eight["exp_avg"], eight["exp_avg_sq"], step=1),
                lambda: learn.adamw_step([x], [x], step=1, betas=(1.0, 0.9), **state),
                lambda: learn.adamw_step([x], [x], step=1, eps=-1.0, **state),
                lambda: learn.AdamW([x]).load_state_dict(learn.AdamW([x, y.float()]).state_dict())):
        with pytest.raises(ValueError):
            bad()
    # a parameter that a later backward pass needs as it was
    w = randn(3, 3, seed=1).requires_grad_(True)
    out = (w * w).sum()
    learn.adamw_step([w], [torch.ones(3, 3, device="cuda")], step=1, **learn.adamw_state([w]))
    with pytest.raises(RuntimeError):
        out.backward()


def test_c_abi_refuses_null_and_malformed_arguments():
    import ctypes as C

    from mymyr_b200.task import default_context

    L, h = _lib.lib(), default_context().handle
    a = _lib.LogprobsArgs()
    assert L.b2_logprobs(None, C.byref(a), None) == _lib.B2_INVALID_ARGUMENT
    assert L.b2_logprobs(h, None, None) == _lib.B2_INVALID_ARGUMENT
    a.temperature, a.rows, a.width = 1.0, 2, 3
    assert L.b2_logprobs(h, C.byref(a), None) == _lib.B2_INVALID_ARGUMENT  # no logits
    a.rows = 1 << 31
    assert L.b2_logprobs(h, C.byref(a), None) == _lib.B2_INVALID_ARGUMENT
    a.rows, a.dtype = 0, 7
    assert L.b2_logprobs(h, C.byref(a), None) == _lib.B2_INVALID_ARGUMENT
    assert L.b2_logprobs_backward(h, C.byref(a), None, None, None, 0, None) == _lib.B2_INVALID_ARGUMENT
    e = _lib.EmbeddingArgs()
    assert L.b2_embedding(h, C.byref(e), None, 0, None, None) == _lib.B2_INVALID_ARGUMENT  # no token width
    e.token_bits, e.count, e.vocabulary, e.width = 64, 5, 3, 4
    assert L.b2_embedding(h, C.byref(e), None, 0, None, None) == _lib.B2_INVALID_ARGUMENT
    t = torch.zeros(64, dtype=torch.int64, device="cuda")
    e.tokens = t.data_ptr()
    assert L.b2_embedding_backward(h, C.byref(e), t.data_ptr(), 4, t.data_ptr(), t.data_ptr(), 16,
                                   None) == _lib.B2_CAPACITY
    w = _lib.AdamwArgs()
    w.count = 1
    assert L.b2_adamw(h, C.byref(w), None) == _lib.B2_INVALID_ARGUMENT
    table = (_lib.AdamwTensor * 1)((t.data_ptr(), t.data_ptr(), 64, 5, 0))
    w.tensors, w.moment_bits, w.step, w.blocks = C.addressof(table), 32, 1, 5
    assert L.b2_adamw(h, C.byref(w), None) == _lib.B2_INVALID_ARGUMENT  # moments outside the arrays
    assert b"" != _lib.last_error().encode()


def test_actions_of_an_expansion():
    """The successors of rl.expand as rows of actions: the log-probability of an action under equal logits is minus the
    log of the state's successor count."""
    task = Task.from_text(tasks.sliding_tile(3, 3, 20, 0))
    env = rl.BatchedEnv(task, 64, seed=1)
    env.reset()
    for _ in range(5):
        env.step()
    e = rl.expand(task, env.states)
    got = learn.logprobs(torch.zeros(e.generated, device="cuda"), torch.zeros(64, dtype=torch.int64, device="cuda"),
                         offsets=e.offsets, top=4)
    count = (e.offsets[1:] - e.offsets[:-1]).double()
    near(got.logprob, -count.log(), 8 * EPS)
    near(got.entropy, count.log(), 8 * EPS)
    assert torch.equal((got.top_tokens >= 0).sum(1), count.long())


def test_gradients_of_gradients_are_refused():
    x, w = randn(4, 50, seed=1).requires_grad_(True), randn(9, 6, seed=2).requires_grad_(True)
    y = some_tokens(4, 50, 3)
    for out, leaf in ((learn.logprobs(x, y).entropy.sum(), x),
                      (learn.embedding(y.clamp(max=8), w).square().sum(), w)):
        g, = torch.autograd.grad(out, leaf, create_graph=True)
        with pytest.raises(RuntimeError, match="differentiable once"):
            g.sum().backward()


def test_inputs_changed_in_place_are_seen():
    x, y = randn(4, 50, seed=1), some_tokens(4, 50, 3)
    leaf = x.clone().requires_grad_(True)
    moved = leaf * 1.0
    out = learn.logprobs(moved, y).logprob.sum()
    with torch.no_grad():
        moved.mul_(2.0)
    with pytest.raises(RuntimeError):
        out.backward()
    t = torch.tensor([1, 2], device="cuda")
    rows = learn.embedding(t, randn(5, 3, seed=1).requires_grad_(True)).sum()
    t.zero_()
    with pytest.raises(RuntimeError):
        rows.backward()
