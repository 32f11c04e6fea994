"""The distillation loss and its gradient against the definition in 64 bits, with
room for what the roundings of one element amount to and no more: a group of
eight that is missing or doubled fails, whatever the length of the row.

EPS is half a step of fp32 (2^-24).  With D = (maximum - x) / tau, the exponent
of an element is a difference, a factor and a product (3 EPS D), taken once more
between the maximum of the others and the row's (EPS D), the exponential is good
to a step (2 EPS); sums pass an element through ``_additions`` roundings.  All of
it is relative to the terms that make an element of the gradient, q and p; the
types' own rounding follows once.
"""
import math

import pytest
import torch

from test_top_distill_beam import DTYPES, EPS, HALF, _dev, _gen, _logits
from test_top_distill_beam import _weights, gpu, ref_distill


def _additions(vocab):
    """Roundings between an element and the sum over its row: the additions of a
    thread (the rows that are read twice: and the rescalings, a few per group),
    of the lanes, of the waves, of the two parts."""
    groups = max(4, -(-vocab // 8192))
    return 8 * groups + 5 * groups + 6 + 16 + 2


def _share(x, mask=None):
    """(softmax along the last axis, log of the sum relative to the maximum, the
    maximum): 0, -inf and 0 where nothing is above -inf."""
    if mask is not None:
        x = torch.where(mask, x, -math.inf)
    high = x.amax(-1, keepdim=True)
    high = torch.where(high == -math.inf, 0.0, high)
    lse = torch.logsumexp(x - high, -1, keepdim=True)
    gone = lse == -math.inf
    return (torch.where(gone, 0.0, (x - high - torch.where(
        gone, 0.0, lse)).exp()), lse, high)


class Exact:
    """loss, grad: the definition (no index twice); loss_tol, grad_tol: see
    above, before the rounding to the gradient's own type."""

    def __init__(self, logits, values, indices, rest, tau, targets=None,
                 lengths=None, hard=0.0):
        steps, batch, vocab = logits.shape
        w = _weights(steps, batch, lengths, None)
        x = torch.where((w > 0)[..., None], logits.double(), 0.0)
        there = (indices >= 0) & (indices < vocab)
        at = torch.where(there, indices, 0).long()
        held = torch.zeros(x.shape).scatter_add_(-1, at, there.float()) > 0
        # (differences to a maximum first: masks of the type's lowest value)
        q, z, top = _share(x / tau)
        others, zo, top_o = _share(x / tau, ~held)
        zo = zo + (top_o - top) - z
        u = torch.where(there, values.double() / tau, -math.inf)
        last = torch.full(w.shape, -math.inf, dtype=torch.float64) \
            if rest is None else rest.double()
        u = torch.cat([u, last[..., None]], -1)
        p, n, top_u = _share(u)
        logq = torch.cat([(x / tau).gather(-1, at) - top - z, zo], -1)
        terms = torch.where(p > 0, p * (u - top_u - n - logq), 0.0)
        kl = terms.sum(-1)
        # a row without any teacher probability has no distillation term
        taught = (u > -math.inf).any(-1, keepdim=True) & (hard < 1)
        kl = torch.where(taught[..., 0], kl, 0.0)
        teacher = torch.zeros_like(x).scatter_add_(
            -1, at, torch.where(there, p[..., :-1], 0.0))
        teacher = torch.where(held, teacher, p[..., -1:] * others)
        soft = (1 - hard) * tau
        row = soft * tau * kl
        grad = torch.where(taught, soft * (q - teacher), 0.0)
        # roundings, relative
        high = x.amax(-1, keepdim=True)
        far = torch.where(x == -math.inf, 0.0, (high - x) / tau)
        adds = _additions(vocab)
        sums = EPS * (adds + 4 + 4 * (q * far).sum(-1, keepdim=True) +
                      4 * (others * far).sum(-1, keepdim=True))
        # (the teacher's exponents: of differences too, those that count)
        wide = (p * torch.where(p > 0, top_u + n - u, 0.0)).sum(-1)
        said = EPS * (8 * wide + 64 + 16)[..., None]
        own = EPS * (4 * far + 8)
        each = torch.zeros_like(x).scatter_add_(-1, at, torch.where(
            there, 4 * EPS * (p * torch.where(p > 0, top_u + n - u, 0.0))
            [..., :-1], 0.0))
        self.grad_tol = soft * ((own + sums) * q + each +
                                (own + sums + said) * teacher)
        # What moves every d = log q - log p by the same is met by sum (q - p) = 0
        # but for the roundings; the rest is relative to the terms, which are not
        # negative
        outcomes = torch.cat([q.gather(-1, at) * there,
                              zo.exp()], -1)
        eps = (sums + said)[..., 0] + EPS * 8
        apart = (outcomes - p).abs().sum(-1)
        kl_tol = 2 * eps * (apart + kl.abs().nan_to_num(0, 0, 0)) + 2 * eps ** 2
        self.loss_tol = soft * tau * kl_tol
        if hard:
            tg = targets.clamp(0, vocab - 1)[..., None]
            s, zh, top = _share(x)
            ce = (zh - (x.gather(-1, tg) - top))[..., 0]
            row = row + hard * ce
            one = torch.zeros_like(x).scatter_(-1, tg, 1.0)
            grad = grad + hard * (s - one)
            sums = EPS * (adds + 4 + 8 * (s * far * tau).sum(-1, keepdim=True))
            self.grad_tol = self.grad_tol + hard * (
                (EPS * (4 * far * tau + 8) + sums) * s + 4 * EPS * one)
            self.loss_tol = self.loss_tol + hard * (
                sums[..., 0] + 4 * EPS * (1 + ce.abs()))
        self.loss = (w * torch.where(w > 0, row, 0.0)).sum()
        self.grad = w[..., None] * grad
        self.grad_tol = w[..., None] * self.grad_tol
        self.loss_tol = float((w * self.loss_tol).sum() +
                              2 * EPS * abs(self.loss))

    def check(self, loss, grad, factor=1.0):
        if loss is not None:
            assert abs(float(loss) - float(self.loss)) <= self.loss_tol
        assert bool(self.fine(grad, factor).all())

    def fine(self, grad, factor=1.0):
        """Which elements of a gradient, times ``factor``, are right."""
        dtype = grad.dtype
        want, tol = self.grad * factor, self.grad_tol * abs(factor)
        tol = tol + 2 * EPS * want.abs()
        # (results of an exponential below 2^-126 are 0)
        tiny = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps / 2
        tol = tol + HALF[dtype] * (want.abs() + tol) + tiny + 2.0 ** -125
        return (grad.double() - want).abs() <= tol


def _case(T, B, V, k, dtype, kind, rest, g, tau=2.0, absent=True):
    logits = _logits((T, B, V), kind, dtype, g)
    teacher = logits.float().clamp(-1e4, 1e4) * 0.7 \
        + torch.randn(T, B, V, generator=g)
    values, indices = torch.topk(teacher, k, dim=-1)
    others = teacher.scatter(-1, indices, -math.inf)
    rest_t = torch.logsumexp(others / tau, -1).float() if rest else None
    indices = indices.int()
    if absent and k > 1:
        keep = torch.randint(1, k + 1, (T, B, 1), generator=g)
        indices = torch.where(torch.arange(k) < keep, indices, -1).int()
    return logits, values.to(dtype), indices, rest_t


def _teacher(values, indices, rest, tau):
    import paccmann_chemistry_amd as P
    dev = _dev()
    return P.TopLogits(values.to(dev), indices.to(dev),
                       None if rest is None else rest.to(dev), tau)


SHAPES = [
    (3, 5, 60, 8, 'normal', True, 0.5), (2, 3, 64, 64, 'ties', False, 0.0),
    (2, 3, 129, 5, 'normal', True, 0.25), (2, 2, 601, 64, 'far', True, 0.25),
    (1, 3, 2050, 17, 'normal', True, 0.0), (2, 2, 5003, 33, 'normal', True, .5),
    (1, 2, 9001, 9, 'masked', True, 0.0), (1, 2, 33001, 64, 'normal', True, .25),
    (1, 2, 32769, 3, 'far', True, 0.5), (1, 2, 50021, 64, 'normal', True, 0.25),
    (1, 2, 50945, 8, 'normal', False, 0.0), (1, 2, 65537, 9, 'normal', True, .5),
    (1, 1, 140001, 9, 'normal', True, 0.5),
]


def _inputs(shape, dtype):
    T, B, V, k, kind, rest, hard = shape
    g = _gen(T, B, V, k, 31)
    case = _case(T, B, V, k, dtype, kind, rest, g)
    targets = torch.randint(0, V, (T, B), generator=g)
    return case, targets


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_the_check_sees_a_group_of_eight(shape, dtype):
    """The exact gradient, rounded, passes; with eight neighbours that are no
    listed tokens 0, doubled or of the next row it does not."""
    (logits, values, indices, rest), targets = _inputs(shape, dtype)
    exact = Exact(logits, values, indices, rest, 2.0, targets, None, shape[-1])
    good = exact.grad.to(dtype)
    assert bool(exact.fine(good).all())
    V = shape[2]
    seen = 0
    for start in range(0, V - 7, max(8, V // 64 // 8 * 8)):
        group = slice(start, start + 8)
        # 16 bits cannot tell what is below their smallest step from 0
        step = torch.finfo(dtype).smallest_normal * torch.finfo(dtype).eps
        if float(good[0, 0, group].abs().max()) < 4 * step:
            continue
        seen += 1
        for factor in (0, 2):
            bad = good.clone()
            bad[0, 0, group] *= factor
            assert not bool(exact.fine(bad).all()), (start, factor)
    assert seen or shape[4] == 'far'


def test_two_ways_to_the_definition():
    """The closed form above against autograd through the definition."""
    g = _gen(3, 4)
    logits, values, indices, rest = _case(2, 3, 40, 6, torch.float32, 'normal',
                                          True, g)
    targets = torch.randint(0, 40, (2, 3), generator=g)
    lengths = torch.tensor([2, 1, 2])
    exact = Exact(logits, values, indices, rest, 2.0, targets, lengths, 0.3)
    loss, grad = ref_distill(logits, values, indices, rest, 2.0, targets,
                             lengths, 0.3)
    assert abs(loss - exact.loss) < 1e-13
    assert bool(((grad - exact.grad).abs() < 1e-14).all())


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shape', SHAPES)
def test_distill_element_by_element(shape, dtype):
    import paccmann_chemistry_amd as P
    (logits, values, indices, rest), targets = _inputs(shape, dtype)
    hard = shape[-1]
    exact = Exact(logits, values, indices, rest, 2.0, targets, None, hard)
    x = logits.to(_dev()).requires_grad_(True)
    loss = P.distill_loss(x, _teacher(values, indices, rest, 2.0),
                          targets=targets.to(_dev()), hard_weight=hard)
    grad, = torch.autograd.grad(loss, x)
    exact.check(loss.detach(), grad.cpu())


def _full_list(V, k, shift, tau, kind, dtype):
    """Rows whose list holds every token that is above -inf, far from 0."""
    g = _gen(V, k, shift, tau * 1000)
    T, B = 2, 3
    logits = torch.full((T, B, V), -math.inf)
    places = torch.rand(T, B, V, generator=g).topk(k, -1).indices
    said = torch.randn(T, B, k, generator=g) * tau
    near = said + torch.randn(T, B, k, generator=g) * tau
    logits.scatter_(-1, places, near + shift)
    rest = torch.full((T, B), -math.inf) if kind == 'empty' else None
    return (logits.to(dtype), said.to(dtype), places.int(), rest,
            places[..., k // 2])


FULL = [(20, 20), (60, 60), (64, 64), (60, 7), (300, 9), (900, 64), (5000, 9),
        (40001, 33), (70001, 9)]


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('shift,tau', [(0, 1.0), (-100, 1.0), (-300, 1.0),
                                       (-12, 0.1), (-20, 0.1), (-2, 0.004),
                                       (300, 1.0)])
@pytest.mark.parametrize('V,k', FULL)
def test_distill_where_no_other_token_is_left(V, k, shift, tau, dtype):
    """A list over the whole vocabulary, or the others masked: their share is 0
    however low the logits are."""
    import paccmann_chemistry_amd as P
    dev = _dev()
    for kind, hard in (('none', 0.0), ('empty', 0.25)):
        logits, values, indices, rest, targets = _full_list(V, k, shift, tau,
                                                            kind, dtype)
        exact = Exact(logits, values, indices, rest, tau, targets, None, hard)
        x = logits.to(dev).requires_grad_(True)
        loss = P.distill_loss(x, _teacher(values, indices, rest, tau),
                              targets=targets.to(dev), hard_weight=hard)
        grad, = torch.autograd.grad(loss, x)
        exact.check(loss.detach(), grad.cpu())
    # a teacher that gives the others probability: infinite, and no NaN
    rest = torch.full(logits.shape[:2], -3.0)
    for hard in (0.0, 0.25):
        loss = P.distill_loss(
            logits.to(dev), _teacher(values, indices, rest, tau),
            targets=targets.to(dev), hard_weight=hard)
        assert float(loss) == math.inf


def test_a_full_list_does_not_change_with_a_shift():
    """... and the definition says so."""
    for V, k in FULL[:5]:
        losses = []
        for shift in (0, -100, -300):
            logits, values, indices, rest, targets = _full_list(
                V, k, 0, 1.0, 'empty', torch.float32)
            exact = Exact(logits + shift, values, indices, rest, 1.0, targets,
                          None, 0.25)
            losses.append(float(exact.loss))
        assert math.isfinite(losses[0]) and losses[0] > 0
        # (32-bit logits, shifted: half a step of 300 each)
        assert max(losses) - min(losses) < 6 * 2.0 ** -15


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('B,V,k,hard', [
    (64, 60, 8, 0.5), (64, 500, 8, 0.0), (64, 1500, 9, 0.25),
    (64, 32000, 32, 0.0), (3, 45001, 64, 0.5), (2, 70001, 9, 0.25)])
def test_distill_gradient_times_a_factor(B, V, k, hard, dtype):
    """The incoming gradient goes in before the gradient is rounded: what 16 bits
    cannot hold without a loss scale they hold with it.  (bf16, which has fp32's
    exponents, is rounded before and after, so twice.)"""
    import paccmann_chemistry_amd as P
    g = _gen(B, V, k)
    logits, values, indices, rest = _case(1, B, V, k, dtype, 'normal', True, g)
    targets = torch.randint(0, V, (1, B), generator=g)
    lengths = (torch.arange(B) != 1).int()
    exact = Exact(logits, values, indices, rest, 2.0, targets, lengths, hard)
    dev = _dev()
    x = logits.to(dev)
    x[0, 1] = math.nan
    x.requires_grad_(True)
    teacher = _teacher(values, indices, rest, 2.0)
    wide = _strided_leaf(x.detach(), dev)
    for leaf in (x, wide):
        for factor in (1.0, 1024.0, 65536.0, -0.25):
            loss = P.distill_loss(leaf, teacher, targets=targets.to(dev),
                                  lengths=lengths.to(dev), hard_weight=hard)
            grad, = torch.autograd.grad(loss * factor, leaf)
            got = grad.cpu()
            assert got.dtype == dtype
            fine = exact.fine(got, factor)
            if dtype == torch.bfloat16:
                fine |= (got.double() - exact.grad * factor).abs() <= \
                    exact.grad_tol * abs(factor) + \
                    2.01 * HALF[dtype] * (exact.grad * factor).abs()
            assert bool(fine.all())
            assert bool((got[0, 1] == 0).all())


def _strided_leaf(x, dev):
    """A leaf whose rows are 3 elements further apart."""
    wide = torch.full(x.shape[:-1] + (x.shape[-1] + 3, ), math.nan,
                      dtype=x.dtype, device=dev)
    view = wide[..., 1:-2]
    view.copy_(x)
    return view.detach().requires_grad_(True)


@gpu
def test_distill_of_half_precision_more_than_once():
    """fp16: the gradient is made in the backward call, so a graph that is kept
    gives it again, and logits that changed meanwhile raise."""
    import paccmann_chemistry_amd as P
    g = _gen(41)
    dev = _dev()
    for V in (60, 900):
        logits, values, indices, rest = _case(3, 4, V, 6, torch.float16,
                                              'normal', True, g)
        teacher = _teacher(values, indices, rest, 2.0)
        weight = torch.tensor([0.5, 0.0, 2.0], device=dev)
        x = logits.to(dev).requires_grad_(True)
        want, = torch.autograd.grad(
            P.distill_loss(x, teacher, step_weight=weight) * 512.0, x)
        # with one over the rows for a weight it is the weighted one divided
        plain, = torch.autograd.grad(P.distill_loss(x, teacher) * 1024.0, x)
        assert bool(((want[2].double() - plain[2].double() * 4).abs() <= 2.02 *
                     HALF[torch.float16] * want[2].double().abs() + 2.0 ** -22)
                    .all())
        assert bool((want[1] == 0).all())
        loss = P.distill_loss(x, teacher, step_weight=weight) * 512.0
        first, = torch.autograd.grad(loss, x, retain_graph=True)
        again, = torch.autograd.grad(loss, x)
        assert torch.equal(first, want) and torch.equal(again, want)
        with pytest.raises(RuntimeError):
            torch.autograd.grad(loss, x)
        loss = P.distill_loss(x, teacher)
        with torch.no_grad():
            x.mul_(1.0)
        with pytest.raises(RuntimeError, match='inplace operation'):
            loss.backward()


@gpu
@pytest.mark.parametrize('V', [60, 900])
def test_distill_of_half_precision_on_a_side_stream_and_captured(V):
    import paccmann_chemistry_amd as P
    g = _gen(41, V)
    dev = _dev()
    logits, values, indices, rest = _case(3, 4, V, 6, torch.float16, 'normal',
                                          True, g)
    teacher = _teacher(values, indices, rest, 2.0)
    lengths = torch.tensor([3, 1, 2, 3], dtype=torch.int32, device=dev)
    x = logits.to(dev).requires_grad_(True)
    scale = torch.tensor(512.0, device=dev)

    def step(leaf):
        loss = P.distill_loss(leaf, teacher, lengths=lengths)
        return torch.autograd.grad(loss * scale, leaf)[0]
    want = step(x.detach().clone().requires_grad_(True))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        grad = step(x)
    for i, factor in enumerate((512.0, 64.0, 512.0)):
        new = torch.randn(3, 4, V, generator=_gen(i, V)).half().to(dev)
        scale.fill_(factor)
        with torch.no_grad():
            x.copy_(new)
        graph.replay()
        torch.cuda.synchronize()
        eager = step(new.clone().requires_grad_(True))
        torch.cuda.synchronize()
        assert torch.equal(grad, eager)


@gpu
@pytest.mark.parametrize('V', [60, 900, 70001])
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('said', DTYPES)
def test_distill_of_a_teacher_of_another_type(V, dtype, said):
    import paccmann_chemistry_amd as P
    g = _gen(V, 8)
    logits, values, indices, rest = _case(2, 3, V, 7, dtype, 'normal', True, g)
    values = values.to(said)
    exact = Exact(logits, values, indices, rest, 2.0)
    x = logits.to(_dev()).requires_grad_(True)
    loss = P.distill_loss(x, _teacher(values, indices, rest, 2.0))
    grad, = torch.autograd.grad(loss, x)
    exact.check(loss.detach(), grad.cpu())


@gpu
@pytest.mark.parametrize('dtype', [torch.bfloat16, torch.float16])
def test_distill_offsets_beyond_32_bits(dtype):
    """2.15e9 logits, of which the rows at the end take part: what they give by
    themselves, and zeros before them."""
    import paccmann_chemistry_amd as P
    dev = _dev()
    T, B, V, k = 2, 4100, 262144, 5
    x = torch.empty(T, B, V, dtype=dtype, device=dev)
    x.fill_(math.nan)
    g = _gen(V)
    mine = (torch.randn(T, 1, V, generator=g) * 3).to(dtype).to(dev)
    x[:, -1:] = mine
    places = torch.randint(0, V, (T, B, k), generator=g).int().to(dev)
    values = torch.randn(T, B, k, generator=g).to(dev)
    rest = torch.ones(T, B, device=dev)
    targets = torch.randint(0, V, (T, B), generator=g).to(dev)
    lengths = torch.zeros(B, dtype=torch.int32, device=dev)
    lengths[-1] = T

    def run(x, s):
        x.requires_grad_(True)
        teacher = P.TopLogits(values[:, s].contiguous(),
                              places[:, s].contiguous(),
                              rest[:, s].contiguous(), 2.0)
        loss = P.distill_loss(x, teacher, targets=targets[:, s].contiguous(),
                              lengths=lengths[s], hard_weight=0.25)
        return loss.detach(), torch.autograd.grad(loss * 64, x)[0]
    want, want_grad = run(mine, slice(B - 1, B))
    loss, grad = run(x, slice(0, B))
    assert torch.equal(loss, want)
    assert torch.equal(grad[:, -1:], want_grad)
    assert not bool(grad[0, :-1].any()) and not bool(grad[1, :-1].any())


@gpu
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
@pytest.mark.parametrize('V', [20, 400, 900, 5000, 70001])
def test_distill_of_a_loss_in_range_whose_parts_are_not(V, dtype):
    """Tokens that the teacher lists and the student masks with its type's lowest
    value, below temperature 1: log q is -1.7e39, tau^2 of it over the batch is a
    32-bit number."""
    import paccmann_chemistry_amd as P
    g = _gen(V, 77)
    logits, values, indices, rest = _case(2, 5, V, 6, dtype, 'normal', True, g,
                                          tau=0.2, absent=False)
    logits.scatter_(-1, indices[..., 2:3].long(), torch.finfo(dtype).min)
    values = torch.randn(values.shape, generator=g).to(dtype) * 0.1
    values[..., 2] = 0.5
    rest.fill_(-1.0)
    exact = Exact(logits, values, indices, rest, 0.2)
    assert 1e36 < float(exact.loss) < 3e38
    x = logits.to(_dev()).requires_grad_(True)
    loss = P.distill_loss(x, _teacher(values, indices, rest, 0.2))
    grad, = torch.autograd.grad(loss, x)
    # (p is off by its exponent's roundings, and the loss by as much of itself)
    assert abs(float(loss.detach()) - float(exact.loss)) <= \
        1e-5 * float(exact.loss)
    assert bool(exact.fine(grad.cpu()).all())


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('tau', [0.02, 0.7, 1.0, 3.0, 900.0])
@pytest.mark.parametrize('V', [20, 400, 900, 5000, 70001])
def test_distill_of_teachers_that_are_far_away(V, tau, dtype):
    """Lists of nothing but the type's lowest value (uniform), with the others at
    -inf, absent or finite; lists near the largest one, and far below their
    rest; what counts is differences."""
    import paccmann_chemistry_amd as P
    g = _gen(V, 78)
    T, B, k = 2, 5, 7
    logits = torch.randn(T, B, V, generator=g).to(dtype)
    indices = torch.rand(T, B, V, generator=g).topk(k, -1).indices.int()
    values = torch.randn(T, B, k, generator=g) * min(tau, 30.0)
    low = torch.finfo(dtype).min
    rest = torch.full((T, B), -math.inf)
    values[0, 0] = low
    values[0, 1] = low
    rest[0, 1] = -2.0
    values[0, 2, 1:] = low
    values[0, 3] = low
    indices[0, 3, 3:] = -1
    values[0, 4] = -low          # all of them at the largest value
    values[1, 0, 3] = -low       # one
    values[1, 1] += 1e4          # (in 32 bits to 1e-3)
    rest[1, 1] = 1e4 / tau
    values[1, 2] -= 1e4
    rest[1, 3] = 88.0
    values[1, 4] = -math.inf
    rest[1, 4] = -1e30
    values = values.to(dtype)
    targets = torch.randint(0, V, (T, B), generator=g)
    exact = Exact(logits, values, indices, rest, tau, targets, None, 0.25)
    assert math.isfinite(float(exact.loss))
    x = logits.to(_dev()).requires_grad_(True)
    for r in (rest, None):
        if r is None:
            exact = Exact(logits, values, indices, r, tau, targets, None, 0.25)
        loss = P.distill_loss(x, _teacher(values, indices, r, tau),
                              targets=targets.to(_dev()), hard_weight=0.25)
        grad, = torch.autograd.grad(loss, x)
        exact.check(loss.detach(), grad.cpu())
