"""Preference loss and gradient (csrc/preference.hip, keras.losses.PreferenceLoss) on the GPU against the plain 64-bit form.

The kernels sum in fp64 and round once to fp32 (the gradient: the coefficient once, times the upstream once more), so a loss or
a gradient is off by 2 U of itself; fp64 roundings, e^x to 1e-15 of them, are counted by 1e-12 of the sums of absolute values."""
import pytest
import torch

from tests import training_ops as T

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def K():
    from ranking_amd.keras import losses
    return losses


def make(B, L, tokens, seed=0, graded=True):
    g = torch.Generator().manual_seed(seed + L + tokens)
    lp = -torch.rand(B, L, tokens, generator=g) * 3
    ref = lp + torch.randn(B, L, tokens, generator=g) * 0.2
    mask = torch.rand(B, L, tokens, generator=g) < 0.7
    y = torch.randint(-1, 4, (B, L), generator=g).float() if graded else torch.tensor([1.0, 0.0]).expand(B, 2).contiguous()
    return y, lp, ref, mask, torch.rand(B, generator=g) + 0.1


def check(y, lp, ref, mask, w, kind='logistic', beta=0.3, smoothing=0.0, normalize=False, reduction='auto'):
    loss = K().PreferenceLoss(reduction=reduction, beta=beta, kind=kind, label_smoothing=smoothing, length_normalized=normalize)
    on = lambda t: None if t is None else t.to(DEV)                        # noqa: E731
    total, grad = loss.loss_and_grad(on(y), on(lp), on(w), reference=on(ref), mask=on(mask))
    B = lp.shape[0]
    # beta and the smoothing are handed over as fp32
    f32 = lambda v: torch.tensor(v, dtype=torch.float32).item()            # noqa: E731
    scale = f32(1.0 / max(1, B)) if reduction != 'sum' else 1.0
    want, want_grad, size = T.preference(y, lp, ref, mask, w, kind, f32(beta), f32(smoothing), normalize, scale)
    slack = 1e-12 * (1 + size.sum()) ** 2
    T.assert_within(grad, want_grad, 2 * T.U * want_grad.abs() + 1e-12 * (1 + size.amax()) + 2.0 ** -149, 'gradient')
    # the lists' losses are rounded once and added in fp32
    T.assert_within(total, want.sum(), (B + 2) * T.U * want.abs().sum() + slack, 'loss')
    p = on(lp).requires_grad_()
    out = loss(on(y), p, on(w), reference=on(ref), mask=on(mask))
    T.assert_within(out, want.sum(), (B + 2) * T.U * want.abs().sum() + slack, 'loss of the autograd path')
    (out * 2.0).backward()
    assert torch.equal(p.grad, grad * 2.0)
    return total, grad


@pytest.mark.parametrize('kind,smoothing', [('logistic', 0.0), ('logistic', 0.1), ('hinge', 0.0), ('squared', 0.0)])
@pytest.mark.parametrize('normalize', [False, True])
@pytest.mark.parametrize('B,L,tokens', [(1, 2, 1), (5, 3, 17), (3, 5, 300), (2, 64, 9)])
def test_kinds(kind, smoothing, normalize, B, L, tokens):
    check(*make(B, L, tokens), kind=kind, smoothing=smoothing, normalize=normalize)


@pytest.mark.parametrize('B,L,tokens', [(1, 1, 5), (7, 2, 255), (2, 2, 8191), (2, 3, 8193), (1, 2, 40001), (300, 2, 64), (3, 2, 0)])
def test_sizes(B, L, tokens):
    check(*make(B, L, tokens))


@pytest.mark.parametrize('B,L,tokens', [(4500, 3, 5), (5001, 2, 1), (4099, 5, 30), (8191, 1, 3)])
def test_many_short_lists(B, L, tokens):
    """So many that a list has a part of a wavefront, the last wavefront some lists too few."""
    check(*make(B, L, tokens), kind='squared', normalize=True)


def test_tokens_beyond_the_caches():
    """8.7 M tokens go past the caches, each list as it is alone; odd rows."""
    B, L, tokens = 11, 3, 264001
    g = torch.Generator(device=DEV).manual_seed(4)
    lp, ref = (torch.randn(B, L, tokens, device=DEV, generator=g) for _ in range(2))
    mask = torch.rand(B, L, tokens, device=DEV, generator=g) < 0.5
    y = torch.tensor([2.0, 0.0, 1.0], device=DEV).expand(B, L)
    loss = K().PreferenceLoss(reduction='sum', length_normalized=True, beta=1.0)
    total, grad = loss.loss_and_grad(y, lp, reference=ref, mask=mask)
    parts = [loss.loss_and_grad(y[k:k + 1], lp[k:k + 1].clone(), reference=ref[k:k + 1].clone(), mask=mask[k:k + 1].clone()) for k in range(B)]
    # fp64 sums in another order, then the same roundings
    want = torch.cat([p[1] for p in parts]).double()
    T.assert_within(grad, want, 2 * T.U * want.abs())
    T.assert_within(total, sum(p[0].double() for p in parts), (B + 1) * T.U * total.double().abs())
    p = lp.requires_grad_()
    loss(y, p, reference=ref, mask=mask).backward()
    assert torch.equal(p.grad, grad)


def test_optional_arguments():
    y, lp, ref, mask, w = make(4, 3, 50)
    check(y, lp, None, None, None)
    check(y, lp, ref, None, None)
    check(y, lp, None, mask, w, reduction='sum')
    loss = K().PreferenceLoss()
    a = loss.loss_and_grad(y.to(DEV), lp.to(DEV), w.unsqueeze(1).to(DEV), mask=mask.float().to(DEV))
    b = loss.loss_and_grad(y.to(DEV), lp.to(DEV), w.to(DEV), mask=mask.to(torch.uint8).to(DEV))
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    a, b = loss.loss_and_grad(y.to(DEV), lp.to(DEV), 2.0), loss.loss_and_grad(y.to(DEV), lp.to(DEV), torch.tensor(2.0, device=DEV))
    assert torch.allclose(a[0], b[0], rtol=4 * T.U) and torch.allclose(a[1], b[1], rtol=4 * T.U)


def test_scores_of_whole_answers():
    """[B, L] log probabilities of whole answers = answers of one token; unreduced losses."""
    y, lp, ref, _, w = make(6, 4, 1)
    loss = K().PreferenceLoss(reduction='none')
    got = loss(y.to(DEV), lp[:, :, 0].to(DEV), w.to(DEV), reference=ref[:, :, 0].to(DEV))
    f32 = torch.tensor(0.1, dtype=torch.float32).item()
    want, _, _ = T.preference(y, lp, ref, None, w, 'logistic', f32, 0.0, False)
    T.assert_within(got, want, 2 * T.U * want.abs() + 1e-12)
    T.assert_within(loss.call(y.to(DEV), lp[:, :, 0].to(DEV)), T.preference(y, lp, None, None, None, 'logistic', f32, 0.0, False)[0],
                    1e-6 * want.abs().max())
    total, grad = K().PreferenceLoss().loss_and_grad(y.to(DEV), lp[:, :, 0].to(DEV))
    assert grad.shape == (6, 4)


def test_masked_places_are_never_used():
    y, lp, ref, mask, w = make(5, 4, 100)
    y[0] = torch.tensor([2.0, -1.0, 0.0, 1.0])
    clean = check(y, lp, ref, mask, w, normalize=True)
    off = ~mask
    off[0, 1] = True                                                       # an answer that is not there
    for bad in (float('nan'), float('inf'), -float('inf')):
        lp2, ref2 = lp.masked_fill(off, bad), ref.masked_fill(off, bad)
        got = K().PreferenceLoss(beta=0.3, length_normalized=True).loss_and_grad(y.to(DEV), lp2.to(DEV), w.to(DEV), reference=ref2.to(DEV), mask=mask.to(DEV))
        assert torch.equal(got[0], clean[0]) and torch.equal(got[1], clean[1])
    assert not got[1][off.to(DEV)].any()


def test_lists_without_pairs_and_empty_answers():
    y, lp, ref, mask, w = make(4, 3, 20)
    y[0], y[1], y[2] = 1.0, -1.0, torch.tensor([-1.0, 3.0, -1.0])          # ties, nothing there, one answer
    y[3] = torch.tensor([2.0, 1.0, 0.0])
    mask[3, 1] = False                                                     # an answer of no tokens
    _, grad = check(y, lp, ref, mask, w, normalize=True)
    assert not grad[:3].any() and not grad[3, 1].any() and grad[3, 0].any()
    total, grad = check(y[:3], lp[:3], ref[:3], mask[:3], w[:3])
    assert total == 0 and not grad.any()
    nan = torch.full_like(y, float('nan'))
    total, grad = K().PreferenceLoss().loss_and_grad(nan.to(DEV), lp.to(DEV))
    assert total == 0 and not grad.any()


def test_large_margins_and_infinities():
    """Margins far beyond what an exponential takes; an infinite log probability of a token that counts."""
    y = torch.tensor([[1.0, 0.0], [1.0, 0.0]])
    lp = torch.tensor([[[-1.0], [-5e4]], [[-5e4], [-1.0]]])
    total, grad = check(y, lp, None, None, None, beta=1.0)
    assert torch.isfinite(grad).all() and grad[0].abs().max() < 1e-30 and grad[1, 0, 0] == -0.5
    lp[1, 0, 0] = -float('inf')
    total, grad = K().PreferenceLoss(beta=1.0).loss_and_grad(y.to(DEV), lp.to(DEV))
    assert total == float('inf') and grad[1, 0, 0] == -0.5


def test_an_answer_of_probability_zero():
    """-inf on either side of a pair: the loss is infinite where the better answer is impossible, and 0 where the worse one is."""
    y = torch.tensor([[1.0, 0.0], [1.0, 0.0], [1.0, 0.0]])
    lp = torch.tensor([[[-1.0], [-float('inf')]], [[-float('inf')], [-1.0]], [[-float('inf')], [-float('inf')]]])
    loss = K().PreferenceLoss(reduction='none', beta=1.0)(y.to(DEV), lp.to(DEV))
    assert loss[0] == 0 and loss[1] == float('inf') and loss[2].isnan()
    _, grad = K().PreferenceLoss(reduction='sum', beta=1.0).loss_and_grad(y.to(DEV), lp.to(DEV))
    assert not grad[0].any() and grad[1].flatten().tolist() == [-1.0, 1.0]


@pytest.mark.parametrize('B,L,tokens', [(3, 2, 33), (2, 4, 700), (2, 2, 9001)])
def test_shifted_tensors(B, L, tokens):
    """Dense tensors that start anywhere: single tokens an access instead of four, the same sums and gradients."""
    y, lp, ref, mask, w = make(B, L, tokens)
    y[:, 0], y[:, 1] = 2.0, 1.0
    want = K().PreferenceLoss().loss_and_grad(y.to(DEV), lp.to(DEV), w.to(DEV), reference=ref.to(DEV), mask=mask.to(DEV))

    def shifted(t):
        flat = torch.zeros(t.numel() + 1, dtype=t.dtype, device=DEV)
        flat[1:] = t.flatten().to(DEV)
        return flat[1:].view(t.shape)
    for move in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 1, 1)):
        a, b, c = (shifted(t) if m else t.to(DEV) for t, m in zip((lp, ref, mask), move))
        got = K().PreferenceLoss().loss_and_grad(y.to(DEV), a, w.to(DEV), reference=b, mask=c)
        # fp64 sums in another order: the same after rounding but for the last bit
        T.assert_within(got[0], want[0].double(), 2 * T.U * want[0].double().abs() + 1e-12)
        T.assert_within(got[1], want[1].double(), 2 * T.U * want[1].double().abs() + 1e-12)


def test_strides_types_and_empty_batch():
    y, lp, ref, mask, w = make(6, 4, 30)
    want = K().PreferenceLoss().loss_and_grad(y[::2, :3].contiguous().to(DEV), lp[::2, :3, 5:].contiguous().to(DEV),
                                              mask=mask[::2, :3, 5:].contiguous().to(DEV))
    got = K().PreferenceLoss().loss_and_grad(y.to(DEV)[::2, :3], lp.to(DEV)[::2, :3, 5:], mask=mask.to(DEV)[::2, :3, 5:])
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    half = lp.to(torch.bfloat16).to(DEV).requires_grad_()
    K().PreferenceLoss()(y.to(DEV), half).backward()
    assert half.grad.dtype == torch.bfloat16
    full = K().PreferenceLoss().loss_and_grad(y.to(DEV), half.detach().float())[1]
    T.assert_within(half.grad, full.double(), T.half(torch.bfloat16) * full.double().abs() + 1e-40)
    total, grad = K().PreferenceLoss().loss_and_grad(torch.zeros(0, 3, device=DEV), torch.zeros(0, 3, 7, device=DEV))
    assert total == 0 and grad.shape == (0, 3, 7)


@pytest.mark.parametrize('tokens', [40, 20000])
def test_other_stream_and_graphs(tokens):
    y, lp, ref, mask, w = (t.to(DEV) for t in make(3, 2, tokens, graded=False))
    loss = K().PreferenceLoss(label_smoothing=0.1)
    step = lambda: loss.loss_and_grad(y, lp, w, reference=ref, mask=mask)   # noqa: E731
    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    graphs = []
    for _ in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for _ in range(3):
        lp.uniform_(-4, 0)
        for g, _ in graphs:
            g.replay()
        want = step()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals():
    y, lp, ref, mask, w = (t.to(DEV) for t in make(4, 3, 5))
    loss = K().PreferenceLoss()
    for bad in (lambda: loss(y[:3], lp), lambda: loss(y, lp[0, 0]), lambda: loss(y, lp, reference=ref[:, :, :4]), lambda: loss(y, lp, mask=mask[:2]),
                lambda: loss(y, lp, w[:3]), lambda: loss(y, lp, y), lambda: loss(y.new_zeros(1, 65), lp.new_zeros(1, 65, 2)),
                lambda: loss(y.new_zeros(1, 0), lp.new_zeros(1, 0, 2)), lambda: K().PreferenceLoss(reduction='none').loss_and_grad(y, lp)):
        with pytest.raises(ValueError):
            bad()


def test_raw_calls():
    """preference_loss, preference_loss_and_grad and preference_grad by themselves, and what they refuse: every tensor has to be
    dense, of the type and shape that the kernels read."""
    from ranking_amd import preference as P
    y, lp, ref, mask, w = (t.to(DEV) for t in make(4, 3, 50))
    total, grad = P.preference_loss_and_grad(lp, y, ref, mask, w, beta=0.3)
    want = K().PreferenceLoss('sum', beta=0.3).loss_and_grad(y, lp, w, reference=ref, mask=mask)
    assert torch.equal(total, want[0]) and torch.equal(grad, want[1])
    loss, coef = P.preference_loss(lp, y, ref, mask.to(torch.uint8), w, beta=0.3)
    assert loss.shape == (4,) and coef.shape == (4, 3)
    assert torch.equal(P.preference_grad(coef, mask, 50), grad)
    up = torch.tensor([1.0, 2.0, 0.0, -1.0], device=DEV)
    assert torch.equal(P.preference_grad(coef, mask, 50, up), grad * up.view(4, 1, 1))       # the kernel rounds this product too
    wide = torch.cat([lp, lp], 2)
    for bad in (dict(log_probs=lp.double()), dict(log_probs=lp.bfloat16()), dict(log_probs=wide[:, :, :50]), dict(log_probs=lp[0]),
                dict(labels=y[:3]), dict(labels=y.long()), dict(labels=y.t().contiguous().t()), dict(reference=ref[:, :, :49].contiguous()),
                dict(reference=ref.half()), dict(mask=mask.float()), dict(mask=mask[:, :2].contiguous()), dict(list_weights=w[:2]),
                dict(list_weights=w.double()), dict(kind='other')):
        for call in (P.preference_loss, P.preference_loss_and_grad):
            with pytest.raises(ValueError):
                call(**dict(dict(log_probs=lp, labels=y, reference=ref, mask=mask, list_weights=w), **bad))
    for bad in ((coef.double(), mask, 50), (coef[0], mask, 50), (coef, mask, 49), (coef, mask.float(), 50), (coef, mask, 50, up[:3]),
                (coef, mask, 50, up.double()), (coef, None, -1), (coef.repeat(1, 22), None, 50)):
        with pytest.raises(ValueError):
            P.preference_grad(*bad)


@pytest.mark.parametrize('B,tokens', [(1, 3), (40001, 2), (2, 9000)])
def test_the_scalar_of_both_paths_and_in_a_graph(B, tokens):
    """At sizes where __call__ and loss_and_grad take the same sums the scalars are the same bits, eager and on every replay."""
    y, lp, ref, mask, w = (t.to(DEV) for t in make(B, 2, tokens, graded=False))
    loss = K().PreferenceLoss(label_smoothing=0.1)
    p = lp.clone().requires_grad_()
    out = loss(y, p, w, reference=ref, mask=mask)
    out.backward()
    total, grad = loss.loss_and_grad(y, lp, w, reference=ref, mask=mask)
    assert out.shape == () and torch.equal(out, total) and torch.equal(p.grad, grad)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.no_grad(), torch.cuda.graph(g):
        held = loss(y, lp, w, reference=ref, mask=mask)
    for _ in range(4):
        lp.uniform_(-4, 0)
        g.replay()
        total, _ = loss.loss_and_grad(y, lp, w, reference=ref, mask=mask)
        torch.cuda.synchronize()
        assert torch.equal(held, total)


@pytest.mark.parametrize('kind', ['logistic', 'hinge', 'squared'])
@pytest.mark.parametrize('tokens', [3, 700, 5000])
def test_nan_of_a_token_is_seen(kind, tokens):
    """A NaN among an answer's tokens makes its list's loss NaN and the gradients of every answer that is paired with it, for every kind;
    other lists and answers without a pair keep theirs."""
    y = torch.tensor([[2.0, 1.0, -1.0], [1.0, 0.0, 0.0], [1.0, 1.0, 0.0]])
    g = torch.Generator().manual_seed(tokens)
    lp = -torch.rand(3, 3, tokens, generator=g)
    good = lp.clone()
    lp[0, 1, tokens // 2] = float('nan')
    lp[2, 0, 0] = float('nan')                                             # paired with answer 2 alone
    loss = K().PreferenceLoss(kind=kind, reduction='none')
    on = lambda t: t.to(DEV)                                               # noqa: E731
    got, want = loss(on(y), on(lp)).cpu(), loss(on(y), on(good)).cpu()
    assert got[0].isnan() and got[2].isnan() and got[1] == want[1] and want.isfinite().all()
    total, grad = K().PreferenceLoss(kind=kind, reduction='sum').loss_and_grad(on(y), on(lp))
    clean = K().PreferenceLoss(kind=kind, reduction='sum').loss_and_grad(on(y), on(good))[1]
    assert total.isnan()
    assert grad[0, :2].isnan().all() and not grad[0, 2].any() and torch.equal(grad[1], clean[1])
    assert grad[2, 0].isnan().all() and grad[2, 2].isnan().all() and torch.equal(grad[2, 1], clean[2, 1])
