"""What the entry points of top logits, distillation, beam selection and state
reordering promise beside their numbers: what they refuse, what autograd is told,
orders among equals, values bit for bit, the paths of the model around them."""
import ctypes
import json
import math

import pytest
import torch
from torch.autograd import forward_ad

from test_top_distill_beam import DTYPES, PARAMS, _check_beam, _dev, _gen
from test_top_distill_beam import _host, _refused, _rows_of, _vae, gpu
from test_top_distill_beam import ref_beam


def _bits(t):
    """``t`` as whole numbers: -0 is not +0, a NaN is its payload."""
    return t.view({2: torch.int16, 4: torch.int32}[t.element_size()])


# --------------------------------------------------------------------------
# distillation
# --------------------------------------------------------------------------
def _small(dtype=torch.float32):
    import paccmann_chemistry_amd as P
    dev = _dev()
    g = _gen(4, 4)
    x = torch.randn(2, 3, 40, generator=g).to(dtype).to(dev)
    values, places = torch.topk(torch.randn(2, 3, 40, generator=g), 5)
    rest = torch.zeros(2, 3, device=dev)
    return x, P.TopLogits(values.to(dev), places.int().to(dev), rest, 2.0)


@gpu
def test_distill_refuses_forward_mode():
    """A tangent that would be lost raises."""
    import paccmann_chemistry_amd as P
    x, teacher = _small()
    with forward_ad.dual_level():
        plain = float(P.distill_loss(x, teacher))
        dual = forward_ad.make_dual(x, torch.ones_like(x))
        with pytest.raises(RuntimeError, match='forward mode'):
            P.distill_loss(dual, teacher)
        with pytest.raises(RuntimeError, match='forward mode'):
            P.distill_loss(dual.clone().requires_grad_(True), teacher)
        rest = forward_ad.make_dual(teacher.rest, torch.ones_like(teacher.rest))
        with pytest.raises(RuntimeError, match='forward mode'):
            P.distill_loss(x, teacher._replace(rest=rest))
    assert plain == float(P.distill_loss(x, teacher))


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
def test_distill_second_derivative_is_not_left_out(dtype):
    """With create_graph the gradient would be a constant: it raises, and the
    loss can be derived once all the same."""
    import paccmann_chemistry_amd as P
    x, teacher = _small(dtype)
    x.requires_grad_(True)
    want, = torch.autograd.grad(P.distill_loss(x, teacher), x)
    loss = P.distill_loss(x, teacher)
    for _ in range(2):
        with pytest.raises(RuntimeError, match='second derivative'):
            torch.autograd.grad(loss, x, create_graph=True)
    loss = P.distill_loss(x, teacher)
    with pytest.raises(RuntimeError, match='second derivative'):
        grad, = torch.autograd.grad(loss, x, create_graph=True)
        (grad.float().pow(2).sum() + x.float().sum()).backward()
    grad, = torch.autograd.grad(loss, x)
    assert torch.equal(grad, want)


def test_distill_grad_refusals():
    """The gradient's own entry refuses what the loss's does."""
    from paccmann_chemistry_amd import _lib
    lib = _lib.load()
    at, _keep = _host()

    def call(logits=at, dtype=2, ld=20, k=3, targets=at, steps=2, vocab=20,
             tau=1.0, hard=0.5, factor=at, dlogits=at, scratch=at):
        return lib.pcm_distill_grad(
            logits, dtype, ld, at, 0, at, None, k, targets, None, None, steps,
            2, vocab, tau, hard, factor, dlogits, scratch, None)
    for what in ('logits', 'factor', 'dlogits', 'scratch'):
        _refused(lib, call(**{what: None}), 'null')
    _refused(lib, call(dtype=3), 'dtype')
    _refused(lib, call(steps=0), 'shape')
    _refused(lib, call(vocab=(1 << 18) + 1, ld=1 << 20), 'shape')
    _refused(lib, call(ld=19), 'row stride')
    _refused(lib, call(k=65), 'k=65')
    _refused(lib, call(tau=1e-4), 'temperature')
    _refused(lib, call(hard=-0.5), 'hard_weight')
    _refused(lib, call(targets=None), 'targets')


# --------------------------------------------------------------------------
# top logits
# --------------------------------------------------------------------------
def test_top_logits_refuses_temperatures_beyond_its_range():
    """Below 1e-30 the factor 1 / temperature leaves 32 bits."""
    from paccmann_chemistry_amd import _lib
    lib = _lib.load()
    at, _keep = _host()
    for tau in (1e-300, 1e-39, 1e-30, 1e30, math.inf, -1.0):
        _refused(lib, lib.pcm_top_logits(at, 0, 2, 20, 20, 3, tau, at, at, at,
                                         None, 0, None), 'temperature')


@gpu
@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,vocab,k', [
    (3, 16, 16), (9000, 13, 13), (3, 60, 60), (9000, 60, 4),
    (9000, 700, 16), (3, 300, 20), (2, 5003, 40), (2, 33001, 64),
    (1, 262144, 50)])
def test_top_logits_values_keep_their_bits(rows, vocab, k, dtype):
    """-0 and NaN come back as they are."""
    import paccmann_chemistry_amd as P
    g = _gen(rows, vocab, k)
    x = torch.where(torch.rand(rows, vocab, generator=g) < 0.5, 0.0, -0.0)
    x[0, 2] = 1.0
    x = x.to(dtype)
    # payloads: quiet NaNs of both signs where fewer numbers are left than asked
    bits = _bits(x)
    odd = {torch.float32: [0x7FC00123, -0x3FFEDC], torch.bfloat16: [
        0x7FC3, -0x3B], torch.float16: [0x7E05, -0x1F9]}[dtype]
    if vocab == k:
        bits[1, 4:] = torch.tensor(odd, dtype=bits.dtype).repeat(vocab)[
            :vocab - 4]
    top = P.top_logits(x.to(_dev()), k)
    at = top.indices.cpu().long()
    assert torch.equal(_bits(top.values.cpu()), bits.gather(1, at))
    if rows > 2:
        assert torch.equal(at[2], torch.arange(k))
    assert at[0, :3].tolist() == [2, 0, 1]


# --------------------------------------------------------------------------
# beam selection
# --------------------------------------------------------------------------
@gpu
@pytest.mark.parametrize('V', [20, 60, 700, 9000])
@pytest.mark.parametrize('lost', [-math.inf, math.nan])
def test_ended_beams_without_a_score(V, lost):
    """A beam that ended and holds nothing: all its candidates are -inf, so they
    are in the order of the tokens, the end token among them."""
    import paccmann_chemistry_amd as P
    g = _gen(V)
    dev = _dev()
    logits = torch.randn(2, 4, V, generator=g)
    scores = torch.tensor([[lost, lost, -1.0, lost], [lost, -2.0, lost, lost]],
                          dtype=torch.float64)
    finished = torch.tensor([[True, True, False, False],
                             [True, True, True, True]])
    for end in (0, 2, 7):
        want = ref_beam(logits, scores, 5, 1.0, finished, end)
        step = P.beam_select(logits.to(dev), scores.to(dev), width=5,
                             finished=finished.to(dev), end_token=end)
        _check_beam(step, want, logits)
    assert want[0][:, 0].tolist() == [0, 1, 2, 3, 4]


@gpu
@pytest.mark.parametrize('V,batch', [(60, 5), (60, 3000), (128, 2), (700, 2),
                                     (5003, 2)])
def test_beams_of_infinite_score(V, batch):
    """A score of +inf (a forced beam) wins with its tokens in order; tokens
    that are masked stay at -inf, and every place is filled."""
    import paccmann_chemistry_amd as P
    dev = _dev()
    logits = torch.full((3, batch, V), -math.inf)
    logits[:, :, 5:8] = torch.tensor([1.0, 3.0, 2.0])
    scores = torch.full((3, batch), -1.0, dtype=torch.float64)
    scores[1] = math.inf
    step = P.beam_select(logits.to(dev), scores.to(dev), width=9)
    inf, low = math.inf, 0.0
    tokens, parents = step.tokens.cpu(), step.parents.cpu()
    # equal sums of one beam: the larger logit first
    assert bool((parents[:3] == 1).all())
    assert bool((tokens[:3] == torch.tensor([[6], [7], [5]])).all())
    assert bool((step.scores.cpu()[:3] == inf).all())
    assert bool((step.scores.cpu()[3:] < low).all())
    assert bool((tokens[3:] == torch.tensor(
        [[6], [6], [7], [7], [5], [5]])).all())
    assert bool((parents[3:] == torch.tensor(
        [[0], [2], [0], [2], [0], [2]])).all())
    step = P.beam_select(logits.to(dev), scores.to(dev), width=12)
    assert bool((step.scores.cpu()[9:] == -inf).all())
    assert bool((step.parents.cpu()[9:] == 0).all())
    assert bool((step.tokens.cpu()[9:] == torch.tensor([[0], [1], [2]])).all())


@gpu
@pytest.mark.parametrize('K,B,V', [(3, 40, 60), (5, 9, 128), (4, 9, 700),
                                   (3, 4, 5003), (2, 3, 32000), (4, 1, 131071),
                                   (2, 2, 200001)])
@pytest.mark.parametrize('scale,tau', [(3.0, 1.0), (0.1, 0.7), (20.0, 2.5)])
def test_beam_scores_have_the_bits_of_their_type(K, B, V, scale, tau):
    """Sums of exponentials in 64 bits all the way.  With u half a step of
    theirs, 2^-53, and D = (maximum - x) / tau: the exponent's factor and the
    temperature's inverse are rounded (2 u D), the exponential is good to a step
    and the remainder's rounding (4 u), a sum passes an element through 8 groups
    of additions at most per 4096 (of a thread; 13 for those of a wave and the
    waves, 64 parts); the score is a difference and a sum."""
    import paccmann_chemistry_amd as P
    g = _gen(K, B, V, scale * 10)
    logits = torch.randn(K, B, V, generator=g) * scale
    scores = -20 * torch.rand(K, B, generator=g, dtype=torch.float64)
    step = P.beam_select(logits.to(_dev()), scores.to(_dev()), temperature=tau)
    x = logits.double() / tau
    far = x.amax(-1, keepdim=True) - x
    lse = torch.logsumexp(x, -1)
    rows = step.parents.cpu().long(), torch.arange(B).expand(K, B)
    at = (*rows, step.tokens.cpu())
    want = scores[rows] + (x[at] - lse[rows])
    u = 2.0 ** -53
    mean = ((x - lse[..., None]).exp() * far).sum(-1)[rows]
    size = x.abs().amax(-1)[rows] + scores[rows].abs() + lse[rows].abs() + 20
    tol = u * (2 * mean + 4 + 8 * max(4, V // 4096) + 13 + 64
               + 2 * far[at] + 4 * size)
    # (the comparison's own rounding is in the last term)
    assert bool(((step.scores.cpu() - want).abs() <= tol).all())


def test_launches_of_too_many_threads_are_refused():
    """A launch has less than 2^32 threads, those of its last block included."""
    from paccmann_chemistry_amd import _lib
    lib = _lib.load()
    at, _keep = _host()

    def beam(beams, batch, vocab):
        return lib.pcm_beam_select(
            at, 1, vocab, at, None, beams, batch, vocab, 1, 1.0, -1, at, at,
            at, None, at, 1 << 60, None)

    def top(rows, vocab):
        return lib.pcm_top_logits(at, 1, rows, vocab, vocab, 3, 1.0, at, at,
                                  at, at, 1 << 60, None)

    def distill(steps, batch, vocab, lengths):
        return lib.pcm_distill_loss(
            at, 1, vocab, at, 0, at, None, 1, None, lengths, None, steps,
            batch, vocab, 1.0, 0.0, at, None, at, None, None)
    _refused(lib, beam(16, 1 << 22, 1025), 'too many')
    # the last block of a launch that is just too long, filled up
    _refused(lib, beam(16, (1 << 24) - 1, 200), 'too many')
    _refused(lib, top((1 << 28) - 1, 200), 'too many')
    _refused(lib, distill((1 << 28) - 1, 1, 200, None), 'too many')
    # the weights of the steps
    _refused(lib, distill(1 << 26, 1, 20, at), 'too many')


# --------------------------------------------------------------------------
# states that follow their beams
# --------------------------------------------------------------------------
@gpu
def test_reorder_states_tells_autograd():
    """What an operation saved of a state before is not silently another."""
    import paccmann_chemistry_amd as P
    dev = _dev()
    parents = torch.tensor([[1, 0], [0, 1]], dtype=torch.int32, device=dev)
    hidden = torch.randn(4, 8, generator=_gen(1)).to(dev)
    stack = torch.randn(2, 4, 3, generator=_gen(2)).to(dev)
    weight = torch.ones(3, 8, device=dev, requires_grad=True)
    out = torch.nn.functional.linear(hidden, weight)
    before = hidden._version, stack._version
    P.reorder_states(parents, [hidden, stack], [0, 1])
    assert (hidden._version, stack._version) == (before[0] + 1, before[1] + 1)
    with pytest.raises(RuntimeError, match='inplace operation'):
        out.sum().backward()
    with torch.inference_mode():
        state = torch.arange(4.0, device=dev).view(4, 1)
        P.reorder_states(parents, [state, hidden])
        assert state.view(-1).tolist() == [2.0, 1.0, 0.0, 3.0]


@gpu
def test_reorder_states_refuses_forward_mode():
    """A tangent that would stay where it was raises."""
    import paccmann_chemistry_amd as P
    dev = _dev()
    parents = torch.tensor([[1], [1]], dtype=torch.int32, device=dev)
    state = torch.randn(2, 8, generator=_gen(1)).to(dev)
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(state, torch.ones_like(state))
        with pytest.raises(ValueError, match='tangent'):
            P.reorder_states(parents, [dual])
        P.reorder_states(parents, [state])
    assert torch.equal(state[0], state[1])


def test_reorder_states_of_interleaved_tensors():
    """Whether tensors share memory is asked of their elements, not of the
    stretch they lie in; the parents count too."""
    from paccmann_chemistry_amd import _lib
    lib = _lib.load()
    at, _keep = _host()
    base = at.value

    def call(states, beams=2, batch=2):
        table = (_lib.PcmState * len(states))(
            *[_lib.PcmState(*s) for s in states])
        return lib.pcm_reorder_states(base + 4096, beams, batch, table,
                                      len(states), None, None)
    # rows of 64 bytes, three columns: overlapping by one byte
    _refused(lib, call([(base, 1, 0, 64, 16), (base + 15, 1, 0, 64, 8)]),
             'another')
    _refused(lib, call([(base + 8, 1, 0, 64, 16), (base, 1, 0, 64, 9)]),
             'another')
    # the second's end meets the next row's beginning
    _refused(lib, call([(base, 1, 0, 64, 16), (base + 48, 1, 0, 64, 17)]),
             'another')
    _refused(lib, call([(base, 1, 0, 64, 16), (base + 32, 2, 128, 32, 16)]),
             'another')
    _refused(lib, call([(base + 4092, 1, 0, 64, 16)]), 'parents')
    _refused(lib, call([(base, 1, 0, 2048, 16)]), 'parents')


@gpu
def test_reorder_states_that_lie_between_each_other():
    import paccmann_chemistry_amd as P
    dev = _dev()
    g = _gen(6)
    K, B = 3, 4
    parents = torch.randint(0, K, (K, B), generator=g, dtype=torch.int32)
    rows = _rows_of(parents)
    pairs = torch.randn(2, K * B, 3, 5, generator=g)
    got = pairs.to(dev)
    P.reorder_states(parents.to(dev), [got[:, :, 0], got[:, :, 2]], 1)
    want = pairs.clone()
    want[:, :, 0] = pairs[:, rows, 0]
    want[:, :, 2] = pairs[:, rows, 2]
    assert torch.equal(got.cpu(), want)
    halves = torch.randn(K * B, 10, generator=g)
    got = halves.to(dev)
    P.reorder_states(parents.to(dev), [got[:, 6:], got[:, :6]])
    assert torch.equal(got.cpu(), halves[rows])
    with pytest.raises(P._lib.PaccmannHipError, match='memory'):
        P.reorder_states(parents.to(dev), [got[:, 5:], got[:, :6]])
    square = torch.randn(K * B, K * B, device=dev)
    with pytest.raises(TypeError, match='list'):
        P.reorder_states(parents.to(dev), square)


# --------------------------------------------------------------------------
# the model's paths
# --------------------------------------------------------------------------
def test_every_search_comes_from_the_params():
    """decoder_search, with the other three keys, as the training script reads
    them; keys that a search does not know are left alone."""
    import paccmann_chemistry_amd as P
    from paccmann_chemistry.utils.hyperparams import search_from_params
    params = {'temperature': 0.7, 'beam_width': 4, 'top_tokens': 6}
    for name, kind in (('sampling', P.SamplingSearch),
                       ('greedy', P.GreedySearch), ('beam', P.BeamSearch),
                       ('joint_beam', P.JointBeamSearch)):
        search = search_from_params(dict(params, decoder_search=name))
        assert type(search) is kind
        for key in ('temperature', 'beam_width', 'top_tokens'):
            assert getattr(search, key, params[key]) == params[key]
    joint = search_from_params({'decoder_search': 'joint_beam'})
    assert (joint.beam_width, joint.temperature) == (3, 1.0)
    assert type(search_from_params({})) is P.SamplingSearch
    with pytest.raises(KeyError):
        search_from_params({'decoder_search': 'widest'})


def test_generation_until_a_token_on_the_device_refusals():
    from paccmann_chemistry_amd import _lib
    lib = _lib.load()
    dims = _lib.make_dims(4, 20, 20, 32, 2, 7, 5, True)
    at, _keep = _host()
    weights = _lib.PcmStackGRUParams()

    def call(end=at, tau=1.0, width=3):
        return lib.pcm_stackgru_generate_joint_beam_until(
            ctypes.byref(dims), ctypes.byref(weights), at, at, None, 0, at, 1,
            4, width, tau, end, at, None, None, at, 0, None, None)
    _refused(lib, call(end=None), 'end token')
    _refused(lib, call(tau=0.0), 'temperature')
    _refused(lib, call(width=17), 'beam_width')


@gpu
def test_joint_beam_search_does_not_wait_for_the_device():
    """An end token on the device is read there."""
    import paccmann_chemistry_amd as P
    vae, _ = _vae(PARAMS, 88)
    vae.eval()
    dev = _dev()
    z = torch.randn(1, 21, 16, generator=_gen(3)).to(dev)
    prime = torch.tensor([2, 7], device=dev)
    search = P.JointBeamSearch(beam_width=3)

    def run(end):
        return vae.decoder.generate_from_latent(z, prime, end, search=search,
                                                generate_len=12)
    free = run(None).cpu()
    first, second = int(free[0, 1]), int(free[5, 3])
    want = {end: run(end) for end in (None, first, second)}
    assert not torch.equal(want[first], want[None])
    ends = {end: torch.tensor([end], device=dev) for end in (first, second)}
    far = torch.tensor([99], device=dev)
    vae.check_tokens()
    torch.cuda.synchronize()
    torch.cuda.set_sync_debug_mode('error')
    try:
        got = {end: run(t) for end, t in ends.items()}
        lost = run(far)
    finally:
        torch.cuda.set_sync_debug_mode('default')
    for end in ends:
        assert torch.equal(got[end], want[end])
    # a token that the vocabulary does not hold ends nothing, and is reported
    assert torch.equal(lost, want[None])
    with pytest.raises(RuntimeError, match='index out of range'):
        vae.check_tokens()
    batches = [torch.randn(1, 21, 16, generator=_gen(i)).to(dev)
               for i in range(4)]
    one = [vae.decoder.generate_from_latent(b, prime, first, search=search,
                                            generate_len=7) for b in batches]
    many = list(P.generate_batches(vae, batches, prime, ends[first],
                                   generate_len=7, search=search))
    assert all(torch.equal(a, b) for a, b in zip(one, many))


def _train(tmp_path, student, teacher, **more):
    import logging
    import os
    from paccmann_chemistry_amd.training import train_vae
    from paccmann_chemistry_amd.utils import collate_fn

    class Language:
        start_index, stop_index = 2, 3
    g = _gen(21)
    data = [torch.randint(4, 37, (int(n), ), generator=g)
            for n in torch.randint(3, 12, (32, ), generator=g)]
    loader = torch.utils.data.DataLoader(data, batch_size=8,
                                         collate_fn=collate_fn, drop_last=True)
    os.makedirs(tmp_path / 'weights', exist_ok=True)
    train_vae(0, student, loader, loader, Language(), str(tmp_path),
              log_interval=2, generate_len=6, batch_mode='packed',
              logger=logging.getLogger('test'), teacher=teacher, teacher_top=4,
              **more)


@gpu
def test_train_vae_leaves_the_teacher_as_it_was(tmp_path):
    """It teaches in eval mode, and every module of it has its mode back."""
    params = dict(PARAMS, batch_size=8, batch_mode='packed')
    student, _ = _vae(params, 5, scale=0.1)
    teacher, _ = _vae(params, 6)
    teacher.train()
    teacher.encoder.eval()
    modes = {n: m.training for n, m in teacher.named_modules()}
    seen = []
    teach = teacher.teach

    def watched(*args, **kwargs):
        seen.append([m.training for m in teacher.modules()])
        return teach(*args, **kwargs)
    teacher.teach = watched
    _train(tmp_path, student, teacher)
    assert len(seen) == 4 and not any(any(s) for s in seen)
    assert modes == {n: m.training for n, m in teacher.named_modules()}
    # a student that is its own teacher goes on training
    _train(tmp_path, student, student)
    assert all(m.training for m in student.modules())
    # and if teaching fails

    def broken(*args, **kwargs):
        raise KeyError('no teacher today')
    teacher.teach = broken
    with pytest.raises(KeyError):
        _train(tmp_path, student, teacher)
    assert modes == {n: m.training for n, m in teacher.named_modules()}


@gpu
def test_train_vae_refuses_a_teacher_of_another_vocabulary(tmp_path):
    params = dict(PARAMS, batch_size=8, batch_mode='packed')
    student, _ = _vae(params, 5, scale=0.1)
    other, _ = _vae(dict(params, vocab_size=41, embedding_size=41), 6)
    with pytest.raises(ValueError, match='vocabulary'):
        _train(tmp_path, student, other)


@gpu
def test_train_vae_reports_what_its_teacher_saw(tmp_path):
    """Token ids that the teacher's encoder does not hold raise, at a save before
    anything is written."""
    import os
    import paccmann_chemistry_amd as P
    params = dict(PARAMS, batch_size=8, batch_mode='packed')
    student, _ = _vae(params, 5, scale=0.1)
    small, _ = _vae(dict(params, vocab_size=20, embedding_size=20), 6)
    whole, _ = _vae(params, 6)
    teacher = P.TeacherVAE(small.encoder, whole.decoder)
    with pytest.raises(RuntimeError, match='index out of range'):
        _train(tmp_path, student, teacher)
    with pytest.raises(RuntimeError, match='index out of range'):
        _train(tmp_path, student, teacher, save_interval=2)
    assert os.listdir(tmp_path / 'weights') == []
    _train(tmp_path, student, whole, save_interval=2)
    assert len(os.listdir(tmp_path / 'weights')) == 1


@gpu
@pytest.mark.parametrize('mode', ['padded', 'packed'])
def test_distill_step_reports_its_most_probable_tokens(mode, monkeypatch):
    """``outputs`` is what a step on the targets alone leaves there, and comes
    from this framework's kernels."""
    params = dict(PARAMS, batch_size=6, batch_mode=mode)
    student, _ = _vae(params, 5)
    dev = _dev()
    g = _gen(9)
    lens = [9, 9, 7, 5, 2, 1]
    seqs = [torch.randint(4, 37, (n, ), generator=g) for n in lens]
    if mode == 'packed':
        enc = torch.nn.utils.rnn.pack_sequence([s.to(dev) for s in seqs])
    else:
        enc = torch.nn.utils.rnn.pad_sequence(seqs).to(dev)
    eps = torch.randn(6, 16, generator=g).to(dev)
    student(enc, enc, enc, eps=eps)
    want = student.decoder.outputs
    top = student.teach(enc, enc, k=5, eps=eps)

    def refused(*args, **kwargs):
        raise AssertionError('a library reduction over the logits')
    monkeypatch.setattr(torch.Tensor, 'argmax', refused)
    student.distill(enc, enc, enc, top, eps=eps)
    got = student.decoder.outputs
    assert got.dtype == want.dtype and torch.equal(got, want)


def test_the_example_reads_the_search_from_its_params():
    """Its default params name a search that there is."""
    import os
    from conftest import ROOT
    from paccmann_chemistry_amd.hyperparams import search_from_params
    with open(os.path.join(ROOT, 'examples',
                           'example_params_synthetic.json')) as fp:
        params = json.load(fp)
    assert search_from_params(params).temperature == params['temperature']
    with open(os.path.join(ROOT, 'examples', 'train_vae_synthetic.py')) as fp:
        assert 'search_from_params(params)' in fp.read()


# --------------------------------------------------------------------------
# streams and graphs
# --------------------------------------------------------------------------
@gpu
def test_split_rows_on_two_streams_and_captured():
    """Long rows of few, whose parts meet in a workspace: at once on two streams,
    and replayed from two graphs between eager calls."""
    import paccmann_chemistry_amd as P
    dev = _dev()
    V = 150001

    def inputs(i):
        g = _gen(i, V)
        return [torch.randn(3, 1, V, generator=g).half().to(dev),
                (-torch.rand(3, 1, generator=g, dtype=torch.float64)).to(dev)]

    def work(x, s):
        top = P.top_logits(x, 40, 2.0)
        step = P.beam_select(x, s, width=5, temperature=0.7)
        return [top.values, top.indices, top.rest, *step[:3]]
    want = [[t.clone() for t in work(*inputs(i))] for i in range(3)]
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    data = [inputs(i) for i in range(3)]
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    got = []
    for i in (0, 1, 2, 1, 0, 2):
        with torch.cuda.stream(streams[len(got) % 2]):
            got.append((i, work(*data[i])))
    torch.cuda.synchronize()
    for i, outs in got:
        assert all(torch.equal(a, b) for a, b in zip(outs, want[i]))
    held = [inputs(0), inputs(1)]
    graphs, outs = [torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()], []
    for graph, h in zip(graphs, held):
        with torch.cuda.graph(graph):
            outs.append(work(*h))
    for i in (2, 0, 1, 2):
        for h, j in zip(held, (i, (i + 1) % 3)):
            for t, new in zip(h, data[j]):
                t.copy_(new)
        graphs[0].replay()
        eager = work(*data[i])
        graphs[1].replay()
        torch.cuda.synchronize()
        for have, j in ((outs[0], i), (outs[1], (i + 1) % 3), (eager, i)):
            assert all(torch.equal(a, b) for a, b in zip(have, want[j]))


@gpu
def test_joint_generation_captured():
    """A whole generation in a graph, replayed for other latents and another end
    token on the device."""
    import paccmann_chemistry_amd as P
    vae, _ = _vae(PARAMS, 88)
    vae.eval()
    dev = _dev()
    prime = torch.tensor([2, 7], device=dev)
    search = P.JointBeamSearch(beam_width=4, temperature=0.9)
    z = torch.randn(1, 21, 16, generator=_gen(3)).to(dev)
    end = torch.tensor([3], device=dev)
    vae.decoder._update_batch_size(21)

    def run(z, end):
        return vae.decoder._generate_joint_beam(z, prime, end, search, 11,
                                                return_beams=True)
    run(z, end)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = run(z, end)
    for i, token in ((4, 3), (5, 9), (4, 9), (6, 3)):
        new = torch.randn(1, 21, 16, generator=_gen(i)).to(dev)
        z.copy_(new)
        end.fill_(token)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(outs, run(new, token)):
            assert torch.equal(a, b)
    vae.check_tokens()
