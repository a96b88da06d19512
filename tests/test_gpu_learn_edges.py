"""The learner's operators where they went wrong once, or could: buffers of the caller's own, empty calls, numbers at the
ends of their range, steps that differ from parameter to parameter, arrays past 2^32 elements.

Tolerances come from the roundings a value goes through, EPS = 2^-24 each (32-bit arithmetic)."""

import ctypes as C

import pytest

torch = pytest.importorskip("torch")

pytestmark = pytest.mark.gpu

from mymyr_b200 import _lib, learn  # noqa: E402
from mymyr_b200.task import default_context  # noqa: E402
from test_gpu_learn import DTYPES, HALF_ULP, TINY, near, plain  # noqa: E402

INF = float("inf")
EPS = 2.0 ** -24


@pytest.fixture(scope="module", autouse=True)
def _need_cuda():
    if not torch.cuda.is_available():
        pytest.skip("no CUDA device")


def randn(*shape, seed=0, scale=1.0):
    return torch.randn(*shape, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda") * scale


# ------------------------------------------------------------------------------------------------ log-probabilities

def c_logprobs(logits, tokens=None, **more):
    """The C ABI's arguments for dense rows; the tensors must outlive them."""
    a = _lib.LogprobsArgs()
    a.logits, a.dtype = logits.data_ptr(), [torch.float32, torch.bfloat16, torch.float16].index(logits.dtype)
    a.rows, a.width, a.row_stride, a.temperature = *logits.shape, logits.stride(0), 1.0
    if tokens is not None:
        a.tokens, a.token_bits = tokens.data_ptr(), 64
    for k, v in more.items():
        setattr(a, k, v.data_ptr() if isinstance(v, torch.Tensor) else v)
    return a


def test_statistics_off_a_16_byte_boundary_are_refused():
    """By the host, before anything is launched."""
    L, h = _lib.lib(), default_context().handle
    x, out, stats = randn(3, 9, seed=1), torch.zeros(3, device="cuda"), torch.zeros(16, device="cuda")
    grad = torch.full_like(x, 7.0)
    for off in (1, 2, 3):
        a = c_logprobs(x, entropy=out, stats=stats[off:])
        assert L.b2_logprobs(h, C.byref(a), None) == _lib.B2_INVALID_ARGUMENT
        assert L.b2_logprobs_backward(h, C.byref(a), None, out.data_ptr(), grad.data_ptr(), 9,
                                      None) == _lib.B2_INVALID_ARGUMENT
    torch.cuda.synchronize()
    assert (out == 0).all() and (grad == 7).all()
    a = c_logprobs(x, entropy=out, stats=stats[4:])
    assert L.b2_logprobs(h, C.byref(a), None) == 0
    torch.cuda.synchronize()
    assert (out > 0).all()


def check_sure_rows(width, rows, least, most):
    """A row of one logit of 0, one of -x and no others that count, in any order: S = 1 + exp(-x). Its one rounding is at
    most EPS, and passes to the log-probability (-log S) and the entropy as it is. exp(-x) itself is off by 4 EPS of its
    value and by the roundings of its exponent, 2 EPS of x each, then the product with x, and the quotient and log by a
    unit or two of their own small value."""
    g = torch.Generator(device="cuda").manual_seed(width)
    i = torch.arange(rows, device="cuda")
    x = torch.full((rows, width), -200.0, device="cuda")
    a = torch.randint(0, width, (rows,), generator=g, device="cuda")
    b = (a + 1 + torch.randint(0, width - 1, (rows,), generator=g, device="cuda")) % width
    x[i, b] = -(least + (most - least) * torch.rand(rows, generator=g, device="cuda"))
    x[i, a] = 0.0
    got = learn.logprobs(x, a, top=1)
    d = -x[i, b].double()
    e = (-d).exp()
    logp = -torch.log1p(e)
    entropy = -logp + e * d / (1 + e)
    assert ((got.logprob.double() - logp).abs() <= EPS * (1 + e * (4 * d + 12))).all()
    assert ((got.entropy.double() - entropy).abs() <= EPS * (1 + e * (d + 1) * (4 * d + 12))).all()
    assert torch.equal(got.top_tokens[:, 0], a)


@pytest.mark.parametrize("width", [2, 20, 40, 128])
def test_logprobs_of_sure_rows_are_right_to_a_rounding_of_their_sum(width):
    check_sure_rows(width, 5000, 7.0, 16.0)


@pytest.mark.parametrize("width,rows", [(200, 5000), (3000, 2000), (70001, 300), (300000, 3)])
def test_logprobs_of_long_sure_rows_are_right_to_a_rounding_of_their_sum(width, rows):
    """Wherever the largest logit stands. It is more than 2^10 (6.94 as a logarithm) ahead of all others, so a thread's
    running reference moves to it, and its own term is exactly one."""
    check_sure_rows(width, rows, 7.0, 41.0)


@pytest.mark.parametrize("width,rows", [(3000, 600), (70001, 100)])
def test_entropy_of_spread_rows(width, rows):
    """Normal logits of deviation 8: a few count. A thread's reference lags behind by at most 2^10, so t holds up to ten
    times s more than it is to: three roundings of that when it moves, 6.93 * 3 EPS; two exponentials of 4 EPS; the
    roundings of exponents (2 EPS of d each, d weighted by its share: below the entropy and one) and of the sums (few
    terms count: six roundings of positive ones)."""
    x = randn(rows, width, seed=width, scale=8.0)
    lp = torch.log_softmax(x.double(), 1)
    want = torch.special.entr(lp.exp()).sum(1)
    h = float(want.max())
    got = learn.logprobs(x).entropy.double()
    assert h < 4
    assert float((got - want).abs().max()) <= EPS * (6.93 * 3 + 8 + 2 * (h + 1) + 6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
@pytest.mark.parametrize("first", [0, 17])
def test_gradient_of_a_vector_without_rows(dtype, first):
    """One offset, so no rows, over a buffer of logits: the gradient is zero all over, not what the memory held."""
    offsets = torch.tensor([first], device="cuda")
    for n in (1, 60, 5001):
        leaf = randn(n, seed=n).to(dtype).requires_grad_(True)
        got = learn.logprobs(leaf, torch.zeros(0, dtype=torch.int64, device="cuda"), offsets=offsets, top=2)
        assert got.entropy.shape == got.logprob.shape == (0,) and got.top_tokens.shape == (0, 2)
        held = torch.full_like(leaf, float("nan"))  # what the allocator is to hand out again
        del held
        g, = torch.autograd.grad(got.entropy.sum() + got.logprob.sum(), leaf)
        assert g.shape == leaf.shape and (g == 0).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("counts", [[3, 0, 2, 2, 4] * 50, [2, 3] * 700, [0, 90, 1, 300] * 60, [1, 2] * 300 + [5000, 7]])
def test_gradient_of_every_ragged_row(dtype, counts):
    """All rows against 64 bits; the last counts put a long row into the layout of short ones."""
    n, width = len(counts), max(counts)
    count = torch.tensor(counts, device="cuda")
    offsets = torch.cat((count.new_zeros(1), count.cumsum(0)))
    total = int(offsets[-1])
    flat = randn(total, seed=total, scale=2.0).to(dtype)
    row = torch.repeat_interleave(torch.arange(n, device="cuda"), count)
    place = torch.arange(total, device="cuda") - offsets[row]
    x = torch.full((n, width), -INF, dtype=torch.float64, device="cuda")
    x[row, place] = flat.double()
    tokens = torch.where(count > 0, count // 2, -1)
    gl, ge = randn(n, seed=1), randn(n, seed=2)
    want = plain(x, tokens, None, 1.0, 6, gl, ge)
    leaf = flat.clone().requires_grad_(True)
    got = learn.logprobs(leaf, tokens, offsets=offsets, top=6)
    assert torch.equal(got.top_tokens, want[3])
    grad, = torch.autograd.grad((got.logprob, got.entropy), leaf, (gl, ge))
    # the bounds of the dense form: the spread's roundings, a chain of sums (of up to 1,250 terms for four lanes)
    tol = EPS * (4 * want[6] + 64 + (1250 if width == 5000 else 0))
    size = gl.abs() + ge.abs() * (want[6] + want[1] + 1)
    p, w = want[5][row, place], want[4][row, place]
    bound = (tol * 4 * size)[row] * p + HALF_ULP[dtype] * w.abs() * 1.01 + 2 * TINY[dtype]
    near(grad, w, bound + 4 * EPS * size[row] * (p + (w != 0)))


@pytest.mark.parametrize("width", [30, 1000, 20000])
def test_logprobs_of_rows_past_2_32_elements(width):
    """Three rows, 2^31 + 8 elements apart: the third starts past 2^32 elements. So do its mask and its gradient."""
    free, _ = torch.cuda.mem_get_info()
    if free < 40 << 30:
        pytest.skip("needs 40 GB")
    apart = 2 ** 31 + 8
    big, wide = (torch.zeros(3, apart, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    allowed = torch.zeros(3, apart, dtype=torch.bool, device="cuda")
    x, mask, grad = big[:, :width], allowed[:, :width], wide[:, :width]
    x.copy_(randn(3, width, seed=width))
    mask.copy_(randn(3, width, seed=width + 1) < 1)
    y = mask.int().argmax(1)
    got = learn.logprobs(x, y, mask=mask, top=3)
    leaf = x.contiguous().requires_grad_(True)
    want = learn.logprobs(leaf, y, mask=mask.contiguous(), top=3)
    assert torch.equal(got.logprob, want.logprob.detach()) and torch.equal(got.entropy, want.entropy.detach())
    assert torch.equal(got.top_tokens, want.top_tokens)
    gl, ge, stats = randn(3, seed=1), randn(3, seed=2), torch.zeros(3, 4, device="cuda")
    logprob, entropy = torch.zeros(3, device="cuda"), torch.zeros(3, device="cuda")
    L, h = _lib.lib(), default_context().handle
    a = c_logprobs(x, y, mask=mask, mask_stride=apart, logprob=logprob, entropy=entropy, stats=stats)
    assert L.b2_logprobs(h, C.byref(a), None) == 0, _lib.last_error()
    assert L.b2_logprobs_backward(h, C.byref(a), gl.data_ptr(), ge.data_ptr(), grad.data_ptr(), apart,
                                  None) == 0, _lib.last_error()
    torch.cuda.synchronize()
    each, = torch.autograd.grad((want.logprob, want.entropy), leaf, (gl, ge))
    assert torch.equal(grad, each)
    assert int(torch.count_nonzero(wide)) == int(torch.count_nonzero(each))


def test_embedding_gradient_of_rows_past_2_32_elements():
    free, _ = torch.cuda.mem_get_info()
    if free < 20 << 30:
        pytest.skip("needs 20 GB")
    big = torch.zeros(3, 2 ** 31 + 8, dtype=torch.bfloat16, device="cuda")
    g = big[:, :96]
    g.copy_(randn(3, 96, seed=1))
    w = torch.zeros(7, 96, dtype=torch.bfloat16, device="cuda", requires_grad=True)
    tokens = torch.tensor([4, 2, 6], device="cuda")
    grad, = torch.autograd.grad(learn.embedding(tokens, w), w, g)
    assert torch.equal(grad[tokens], g) and (grad[[0, 1, 3, 5]] == 0).all()


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


HYPER = dict(lr=1e-2, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def formula(p, g, m, v, step, *, lr, betas, eps, weight_decay):
    """A step in 64 bits but for g * g and v, which overflow where 32 bits do. Returns the parameter, the moments and the
    tolerance of the parameter: a rounding of each product, sum, root and quotient of the part that moves, the decay's."""
    b1, b2 = betas
    size = m.abs() * b1 + g.abs() * (1 - b1)
    m, v = m * b1 + g * (1 - b1), v * b2 + (g.float() * g.float()).double() * (1 - b2)
    den = (v / (1 - b2 ** step)).sqrt() + eps
    new = p * (1 - lr * weight_decay) - lr * (m / (1 - b1 ** step)) / den
    return new, m, v, 4 * EPS * p.abs() + 24 * EPS * lr * size / (1 - b1 ** step) / den


@pytest.mark.parametrize("dtype,grad_dtype", [(torch.float32, torch.float32), (torch.bfloat16, torch.bfloat16),
                                              (torch.float16, torch.float32)])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("master", [False, True])
def test_adamw_takes_no_step_where_the_square_of_a_finite_gradient_is_infinite(dtype, grad_dtype, bits, master):
    """v is infinite there, m / inf is zero: the parameter decays, and its neighbours go on as ever. With 32-bit moments
    it stays so; 8 bits have no infinity to hold v by."""
    params = [randn(n, seed=n).to(dtype) for n in (700, 256, 9)]
    state = learn.adamw_state(params, bits=bits, master=master)
    large = torch.zeros(700, dtype=torch.bool, device="cuda")
    large[[0, 8, 255, 256, 511, 699]] = True
    m, v = torch.zeros(700, dtype=torch.float64, device="cuda"), torch.zeros(700, dtype=torch.float64, device="cuda")
    half = 0.0 if dtype == torch.float32 else torch.finfo(dtype).eps / 2
    for step in (1, 2, 3) if bits == 32 else (1,):
        grads = [randn(p.numel(), seed=10 * step + i, scale=0.1).to(grad_dtype) for i, p in enumerate(params)]
        if step == 1:
            grads[0][large] = torch.tensor([2e19, -2e19, 1e20, 3e38, -3e38, 1e30], device="cuda").to(grad_dtype)
        p = (state["master"][:700] if master else params[0]).double()
        learn.adamw_step(params, grads, step=step, **HYPER, **state)
        new, m, v, tol = formula(p, grads[0].double(), m, v, step, **HYPER)
        assert v[large].isinf().all() and v[~large].isfinite().all() and m.isfinite().all()
        assert torch.equal(new[large], (p * (1 - 1e-2 * 0.1))[large])
        if master:
            assert ((state["master"][:700].double() - new).abs() <= tol).all()
        assert ((params[0].double() - new).abs() <= tol + half * new.abs() * 1.01).all()
        assert all(q.isfinite().all() for q in params)
    if bits == 32:
        assert state["exp_avg_sq"][:700][large].isinf().all() and state["exp_avg"].isfinite().all()
    else:
        assert state["exp_avg_sq"][:700].float().isnan().equal(large)


@pytest.mark.parametrize("master", [False, True])
def test_adamw_8_bit_codes_hold_an_infinite_second_moment_as_nan(master):
    """It stays infinite: the parameter decays and takes no step, on later steps too. A gradient's own NaN is held by the
    first moment and goes on spoiling its parameter."""
    p = randn(512, seed=1)
    state = learn.adamw_state([p], bits=8, master=master)
    want = p.clone()
    for step in range(1, 5):
        g = randn(512, seed=10 + step)
        if step == 1:
            g[7], g[300], g[9] = 2e19, -3e38, float("nan")
        learn.adamw_step([p], [g], step=step, **HYPER, **state)
        want = want * (1 - 1e-2 * 0.1)
        assert p[9].isnan() and torch.cat((p[:9], p[10:])).isfinite().all()
        # two roundings each step (of the factor, of the product), on both sides
        assert all(abs(float(p[i] - want[i])) <= 4 * step * EPS * abs(float(want[i])) for i in (7, 300))
    assert state["exp_avg_sq"].float().isnan().nonzero().flatten().tolist() == [7, 9, 300]


@pytest.mark.parametrize("master", [False, True])
def test_adamw_without_eps_takes_second_moments_below_the_normal_numbers_as_they_are(master):
    """32-bit moments. v is subnormal, of 2^-149 steps: three roundings of it come to the tolerance. Where the gradient is
    zero nothing moves."""
    hyper = dict(lr=1e-2, betas=(0.9, 0.9), eps=0.0, weight_decay=0.0)
    u = torch.rand(600, generator=torch.Generator(device="cuda").manual_seed(1), device="cuda")
    g = (u + 1) * 1e-19 * torch.where(u * 16 % 1 < 0.5, -1.0, 1.0)
    g[::7] = 0.0
    g[5::50] = 1.0  # normal numbers beside them
    p = randn(600, seed=2)
    state, before = learn.adamw_state([p], master=master), p.double()
    learn.adamw_step([p], [g], step=1, master=state.pop("master", None), **hyper, **state)
    zero = torch.zeros(600, dtype=torch.float64, device="cuda")
    live = g != 0
    new, _, _, tol = formula(before, g.double(), zero, zero, 1, **hyper)
    v = 0.1 * g.double() ** 2
    tol = tol + hyper["lr"] * 3 * 2.0 ** -149 / v
    assert float(v[live].min()) < 2.0 ** -126 and float(v[live].min()) > 2.0 ** -140
    assert ((p.double() - new).abs() <= tol)[live].all()
    assert torch.equal(p[~live].double(), before[~live])


def test_adamw_8_bits_hold_second_moments_below_the_normal_numbers_as_zero():
    """Zeros among them stay zero, as they do beside an infinity or a NaN."""
    n = 256 * 5
    g = torch.zeros(n, device="cuda")
    g[:256:2] = 1e-20                       # a block of them and of zeros
    g[256:512] = 1e-25                      # of them alone
    g[512], g[768], g[769] = INF, 2e19, 1e-20  # zeros beside infinities
    g[1024:1030] = 1.0
    g[1100] = 1e-20                         # one beside normal numbers
    p = randn(n, seed=1)
    state = learn.adamw_state([p], bits=8)
    learn.adamw_step([p], [g], step=1, **HYPER, **state)
    code = state["exp_avg_sq"].float()
    bad = torch.zeros(n, dtype=torch.bool, device="cuda")
    bad[[512, 768]] = True
    assert code[bad].isnan().all() and (code[1024:1030] > 0).all()
    assert (torch.cat((code[:1024][~bad[:1024]], code[1030:])) == 0).all()


def test_adamw_takes_any_number_of_empty_tensors():
    """Through the C ABI: a launch's worth of them (1,000) before, after and between tensors with elements."""
    L, h = _lib.lib(), default_context().handle
    for places in ([1000], [0], [999], [3, 2500]):
        params = [randn(300, seed=i) for i in range(len(places))]
        want = [p.clone() for p in params]
        g = randn(300, seed=9)
        state = learn.adamw_state(params)
        table = (_lib.AdamwTensor * 3001)()
        for i, (place, p) in enumerate(zip(places, params)):
            table[place] = _lib.AdamwTensor(p.data_ptr(), g.data_ptr(), 300, 2 * i, 0)
        a = _lib.AdamwArgs()
        a.tensors, a.count, a.moment_bits, a.blocks = C.addressof(table), 3001, 32, 2 * len(places)
        a.exp_avg, a.exp_avg_sq = state["exp_avg"].data_ptr(), state["exp_avg_sq"].data_ptr()
        a.lr, a.beta1, a.beta2, a.eps, a.weight_decay, a.step = 1e-3, 0.9, 0.999, 1e-8, 1e-2, 1
        assert L.b2_adamw(h, C.byref(a), None) == 0, _lib.last_error()
        learn.adamw_step(want, [g] * len(places), step=1, **learn.adamw_state(want))
        assert all(torch.equal(p, q) for p, q in zip(params, want))


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_refuses_a_graph(bits):
    """Its replays would repeat one step's corrections, and with 8 bits its random numbers. Nothing is launched; the step
    outside of the capture is taken as ever, and a graph of the other operators stands."""
    p, g = randn(700, seed=1).requires_grad_(True), randn(700, seed=2)
    before = p.detach().clone()
    state = learn.adamw_state([p], bits=bits)
    opt = learn.AdamW([p], bits=bits)
    p.grad = g
    x = randn(5, 40, seed=3)
    want = learn.logprobs(x).entropy
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = learn.logprobs(x).entropy
        with pytest.raises(ValueError, match="captured"):
            learn.adamw_step([p], [g], step=1, **state)
        with pytest.raises(ValueError, match="captured"):
            opt.step()
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(got, want) and torch.equal(p.detach(), before)
    learn.adamw_step([p], [g], step=1, **state)
    assert not torch.equal(p.detach(), before)


@pytest.mark.parametrize("bits", [32, 8])
def test_adamw_corrects_each_parameter_by_its_own_steps(bits):
    """A parameter whose first gradient comes late moves by the learning rate on its first step, whatever the others'
    count; with weights of one sign of gradient only, m' / sqrt(v') is 1 up to the roundings (8-bit codes: half of 2^-4 of
    the first moment, one of 2^-3 of the second's root, none of which has come in on a first step)."""
    a, b = (torch.zeros(300, device="cuda", requires_grad=True) for _ in range(2))
    opt = learn.AdamW([a, b], lr=1e-2, weight_decay=0.0, bits=bits)
    for step in range(1, 12):
        a.grad = torch.ones_like(a)
        b.grad = torch.full_like(b, -3.0) if step == 11 else None
        opt.step()
    assert float((b.detach() - 1e-2).abs().max()) <= 32 * EPS * 1e-2 + 1e-2 * 1e-8 / 3
    assert opt.steps == 11 and opt.param_steps == [[11, 1]]


def test_adamw_object_with_gradients_now_and_then():
    """As torch's, which counts each parameter's steps; and its state, with and without counts of its own."""
    shapes = [(30, 20), (20,), (300,), (7,)]

    def make():
        params = [randn(*s, seed=i).requires_grad_(True) for i, s in enumerate(shapes)]
        return params, [{"params": params[:3]}, {"params": params[3:], "lr": 3e-3}]

    def give(params, step):
        for i, p in enumerate(params):
            p.grad = None if (step + i) % (i + 1) else randn(*p.shape, seed=100 * step + i)

    mine, groups = make()
    opt = learn.AdamW(groups, lr=1e-2, weight_decay=0.1)
    other, groups = make()
    ref = torch.optim.AdamW(groups, lr=1e-2, weight_decay=0.1)
    steps = 13
    saved = None
    for step in range(1, steps + 1):
        for params, o in ((mine, opt), (other, ref)):
            give(params, step)
            o.step()
        if step == 6:
            saved = opt.state_dict()
            saved["state"] = [{k: t.clone() for k, t in s.items()} for s in saved["state"]]
            at = [p.detach().clone() for p in mine]
    for p, q in zip(mine, other):
        # on both sides a step rounds the parameter four times and its part of up to 10 learning rates 24 times
        tol = 2 * steps * EPS * (4 * float(q.detach().abs().max()) + 24 * 10 * 1e-2)
        assert float((p - q).detach().abs().max()) <= tol
    assert opt.param_steps == [[13, 7, 5], [4]]
    again, groups = make()
    with torch.no_grad():
        for p, x in zip(again, at):
            p.copy_(x)
    late = learn.AdamW(groups, lr=1e-2, weight_decay=0.1)
    late.load_state_dict(saved)
    for step in range(7, steps + 1):
        give(again, step)
        late.step()
    assert all(torch.equal(p, q) for p, q in zip(mine, again)) and late.param_steps == opt.param_steps
    old = {k: v for k, v in saved.items() if k != "param_steps"}
    late.load_state_dict(old)
    assert late.steps == 6 and late.param_steps == [[6, 6, 6], [6]]
    with pytest.raises(ValueError):
        late.load_state_dict(saved | {"param_steps": [[1, 2], [3]]})


def test_adamw_takes_a_tensor_for_a_group_and_not_for_its_rows():
    """A tensor is a list of its rows to Python, views that never have a gradient: nothing was updated."""
    w, b = randn(6, 5, seed=1).requires_grad_(True), randn(5, seed=2).requires_grad_(True)
    before = w.detach().clone(), b.detach().clone()
    opt = learn.AdamW([{"params": w}, {"params": [b]}])
    assert [len(g["params"]) for g in opt.param_groups] == [1, 1] and opt.param_groups[0]["params"][0] is w
    w.grad, b.grad = torch.ones_like(w), torch.ones_like(b)
    opt.step()
    assert (w.detach() != before[0]).all() and (b.detach() != before[1]).all()
    with pytest.raises(ValueError):
        learn.AdamW(w)


def test_adamw_refuses_a_parameter_given_twice():
    """A tied one, say: two entries of a launch would update it at once."""
    w, b = randn(6, 5, seed=1).requires_grad_(True), randn(5, seed=2).requires_grad_(True)
    for params in ([w, b, w], [{"params": [w]}, {"params": [b, w]}]):
        with pytest.raises(ValueError, match="twice"):
            learn.AdamW(params)


# ------------------------------------------------------------------------------------------------ saved tensors

def gradients(x, y, mask, ragged, table, tokens):
    x, table = x.clone().requires_grad_(True), table.clone().requires_grad_(True)
    offsets = torch.tensor([0, 40, 40, 160, 201], device="cuda") if ragged else None
    got = learn.logprobs(x.view(-1) if ragged else x, y[:4] if ragged else y, offsets=offsets,
                         mask=mask.view(-1) if ragged else mask)
    rows = learn.embedding(tokens, table, scale=2.0)
    n = got.entropy.shape[0]

    def actions():
        return torch.autograd.grad((got.logprob, got.entropy), x, (randn(n, seed=5), randn(n, seed=6)))[0]

    def embeddings():
        return torch.autograd.grad(rows, table, randn(*rows.shape, seed=7))[0]

    return actions, embeddings


def saved_cases():
    x, y = randn(67, 3, seed=1), torch.randint(0, 3, (67,), generator=torch.Generator(device="cuda").manual_seed(2),
                                               device="cuda")
    mask = randn(67, 3, seed=3) > -0.8
    return x, y, mask, randn(9, 6, seed=4), (y.repeat(2) * 3 % 9).view(2, 67)


@pytest.mark.parametrize("ragged", [False, True])
def test_saved_tensors_may_come_back_in_another_layout(ragged):
    """Hooks that keep them in another order of memory, two elements apart, or on the host."""
    x, y, mask, table, tokens = saved_cases()
    want = [f() for f in gradients(x, y, mask, ragged, table, tokens)]
    apart = lambda t: torch.stack((t, t), -1)[..., 0]  # noqa: E731
    for pack, unpack in ((lambda t: t.t().contiguous() if t.dim() == 2 else t, lambda t: t.t() if t.dim() == 2 else t),
                         (apart, lambda t: t), (lambda t: t.cpu(), lambda t: t.cuda())):
        with torch.autograd.graph.saved_tensors_hooks(pack, unpack):
            got = gradients(x, y, mask, ragged, table, tokens)
        for f, w in zip(got, want):
            assert torch.equal(f(), w)


@pytest.mark.parametrize("ragged", [False, True])
def test_saved_tensors_that_come_back_as_others_are_refused(ragged):
    """Of another type, another size or on another device: an error on the host, before anything is launched."""
    x, y, mask, table, tokens = saved_cases()

    def half(t):
        return t.half() if t.is_floating_point() else t

    def short(t):
        return t[:-1]

    def narrow(t):
        return t.int() if t.dtype == torch.int64 else t

    def host(t):
        return t.cpu()

    for unpack in (half, short, narrow, host):
        with torch.autograd.graph.saved_tensors_hooks(lambda t: t, unpack):
            actions, embeddings = gradients(x, y, mask, ragged, table, tokens)
        for f in (actions, embeddings) if unpack is not half else (actions,):
            with pytest.raises((RuntimeError, ValueError), match="came back"):
                f()
