"""Refusals and host logic of the embedding, token log probability, preference and AdamW entry points (no GPU): argument checks of
the C ABI before any launch, the Python layer's checks, configurations, and the plain 64-bit forms that the GPU tests compare
with, themselves checked against differences and torch."""
import ctypes

import pytest
import torch

import ranking_amd as ra
from ranking_amd import _lib, embedding, optim, preference
from ranking_amd.keras import layers, losses, model, pipeline
from tests import training_ops as T

one = ctypes.c_void_p(256)


def test_embedding_arguments_are_checked_before_any_launch():
    f = _lib.load().tfr_embedding_lookup
    ok = [one, 8, 10, 8, 0, one, 0, 4, 1, 0, 1.0, one, None]

    def call(**change):
        a = list(ok)
        for k, v in change.items():
            a[int(k[1:])] = v
        return f(*a)
    assert call(a4=3) == -1 and call(a6=2) == -1 and call(a9=3) == -1           # type, id type, combiner
    assert call(a1=7) == -1 and call(a3=0) == -1 and call(a2=-1) == -1          # pitch, dim, rows
    assert call(a2=(1 << 25) + 1) == -1 and call(a7=(1 << 25) + 1) == -1        # too many rows, lookups
    assert call(a8=2) == -1 and call(a8=1 << 24, a7=4, a9=1) == -1              # tokens without a combiner; bags * tokens
    assert call(a0=None) == -1 and call(a5=None) == -1 and call(a11=None) == -1
    assert call(a7=0) == 0                                                      # nothing to look up
    g = _lib.load().tfr_embedding_grad
    assert g(one, 0, one, 0, 4, 1, 0, 1.0, 10, 8, one, None, 0, None) == -1     # no workspace
    need = _lib.load().tfr_embedding_grad_workspace_bytes(10, 8, 4, 1, 0)
    assert need > 0
    assert g(one, 0, one, 0, 4, 1, 0, 1.0, 10, 8, one, one, need - 1, None) == -1
    assert g(one, 0, one, 0, 4, 1, 0, 1.0, 10, 8, one, ctypes.c_void_p(264), need, None) == -1
    assert g(one, 0, one, 0, 4, 1, 0, 1.0, 10, 8, None, one, need, None) == -1
    assert g(one, 0, one, 0, 4, 1, 0, 1.0, 0, 8, None, one, need, None) == 0    # no rows
    assert _lib.load().tfr_embedding_grad_workspace_bytes(10, 8, 4, 2, 0) < 0


def test_token_logprob_arguments_are_checked_before_any_launch():
    f, g = _lib.load().tfr_token_logprob, _lib.load().tfr_token_logprob_grad
    assert f(one, 3, 1, 0, 8, one, 4, 8, 1.0, one, None, None, 0, None) == -1
    assert f(one, 0, 0, 0, 8, one, 4, 8, 1.0, one, None, None, 0, None) == -1
    assert f(one, 0, 4, 0, -8, one, 4, 8, 1.0, one, None, None, 0, None) == -1
    assert f(one, 0, 4, 0, 8, one, 4, 0, 1.0, one, None, None, 0, None) == -1
    assert f(one, 0, 4, 0, 8, one, 1 << 24, 8, 1.0, one, None, None, 0, None) == -1
    for t in (0.0, -1.0, float('nan'), float('inf'), 1e-45):
        assert f(one, 0, 4, 0, 8, one, 4, 8, t, one, None, None, 0, None) == -1
        assert g(one, 0, 4, 0, 8, one, one, one, 4, 8, t, one, None) == -1
    assert f(None, 0, 4, 0, 8, one, 4, 8, 1.0, one, None, None, 0, None) == -1
    assert g(one, 0, 4, 0, 8, one, None, one, 4, 8, 1.0, one, None) == -1
    assert f(one, 0, 1, 0, 8, one, 0, 8, 1.0, one, None, None, 0, None) == 0
    need = _lib.load().tfr_token_logprob_workspace_bytes(1, 1 << 20)
    assert need > 0 and f(one, 0, 1, 0, 8, one, 1, 1 << 20, 1.0, one, None, one, need - 1, None) == -1
    assert _lib.load().tfr_token_logprob_workspace_bytes(100000, 100) == 0


def test_preference_arguments_are_checked_before_any_launch():
    f, g = _lib.load().tfr_preference_loss_f32, _lib.load().tfr_preference_grad_f32
    need = _lib.load().tfr_preference_workspace_bytes(2, 3, 5)

    def call(B=2, L=3, T_=5, kind=0, beta=0.1, smoothing=0.0, ws=one, n=need, lp=one):
        return f(lp, None, None, one, None, B, L, T_, kind, beta, smoothing, 0, 1.0, one, one, ws, n, None)
    assert call(L=65) == -1 and call(L=0) == -1 and call(kind=3) == -1 and call(T_=-1) == -1
    assert call(beta=0.0) == -1 and call(beta=float('nan')) == -1 and call(beta=float('inf')) == -1
    assert call(smoothing=0.5) == -1 and call(smoothing=-0.1) == -1
    assert call(ws=None) == -1 and call(n=need - 1) == -1 and call(ws=ctypes.c_void_p(260)) == -1 and call(lp=None) == -1
    assert call(B=0) == 0
    assert g(None, None, None, 2, 3, 5, one, None) == -1 and g(one, None, None, 2, 3, 0, None, None) == 0
    assert _lib.load().tfr_preference_workspace_bytes(1 << 24, 2, 1) < 0
    h = _lib.load().tfr_preference_total_f32
    assert h(None, 2, one, None) == -1 and h(one, 2, None, None) == -1 and h(one, -1, one, None) == -1 and h(one, 1 << 24, one, None) == -1
    assert h(ctypes.c_void_p(260), 2, one, None) == -1


def test_adamw_arguments_are_checked_before_any_launch():
    lib = _lib.load()
    ptr, size = (ctypes.c_void_p * 1)(256), (ctypes.c_int64 * 1)(4)

    def call(dtype=0, count=1, p=ptr, n=size, b1=0.9, b2=0.999, step=1):
        return lib.tfr_adamw(dtype, count, p, ptr, ptr, ptr, n, 1e-3, b1, b2, 1e-8, 0.0, step, None, None)
    assert call(dtype=5) == -1 and call(count=0) == -1 and call(count=89) == -1 and call(p=None) == -1
    assert call(b1=1.0) == -1 and call(b2=float('nan')) == -1 and call(step=0) == -1
    assert call(p=(ctypes.c_void_p * 1)(None)) == -1 and call(n=(ctypes.c_int64 * 1)(-1)) == -1
    assert call(n=(ctypes.c_int64 * 1)(1 << 40)) == -1
    assert call(n=(ctypes.c_int64 * 1)(0)) == 0
    odd = (ctypes.c_void_p * 1)(260)
    assert lib.tfr_adamw8(0, 1, ptr, ptr, odd, ptr, ptr, ptr, size, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, None) == -1
    assert lib.tfr_adamw8(0, 1, ptr, ptr, ptr, None, ptr, ptr, size, 1e-3, 0.9, 0.999, 1e-8, 0.0, 1, None, None) == -1
    assert lib.tfr_adamw_dequantize(one, one, 100, 0, one, None) == -1
    assert lib.tfr_adamw_advance(None, None, 1e-3, 0.9, 0.999, 0.0, one, None) == -1


def test_cpu_tensors_are_refused():
    x = torch.zeros(4, 8)
    ids = torch.zeros(3, dtype=torch.int64)
    with pytest.raises(_lib.TfrHipError):
        embedding.embedding_lookup(x, ids)
    with pytest.raises(_lib.TfrHipError):
        embedding.embedding_grad(x, ids, 4)
    with pytest.raises(_lib.TfrHipError):
        preference.token_log_probs(x, torch.zeros(4, dtype=torch.int64))
    with pytest.raises(_lib.TfrHipError):
        losses.PreferenceLoss()(x, x)
    with pytest.raises(_lib.TfrHipError):
        optim.adamw_step([x], [x], [x], [x], step=1, lr=1e-3)
    with pytest.raises(_lib.TfrHipError):
        optim.dequantize_exp_avg(torch.zeros(128, dtype=torch.int8), torch.zeros(1))


def test_raw_preference_calls_refuse_cpu_tensors():
    from ranking_amd import _lib, preference
    lp, y = torch.zeros(2, 3, 4), torch.zeros(2, 3)
    for bad in (lambda: preference.preference_loss(lp, y), lambda: preference.preference_loss_and_grad(lp, y), lambda: preference.preference_grad(y, None, 4)):
        with pytest.raises(_lib.TfrHipError):
            bad()
    for bad in (lambda: preference.preference_loss(lp, y, kind='other'), lambda: preference.preference_loss_and_grad(lp, y, kind=None)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize('kw', [dict(lr=-1.0), dict(betas=(1.0, 0.9)), dict(betas=(0.9, -0.1)), dict(eps=-1.0), dict(weight_decay=-1.0),
                                dict(state_bits=16), dict(lr=torch.tensor(0.1))])
def test_adamw_hyperparameters(kw):
    with pytest.raises(ValueError):
        optim.AdamW([torch.nn.Parameter(torch.zeros(3))], **kw)


def test_adamw_step_lists():
    with pytest.raises(ValueError):
        optim.adamw_step([], [torch.zeros(1)], [], [], step=1, lr=1e-3)
    with pytest.raises(ValueError):
        optim.adamw_step([], [], [], [], step=0, lr=1e-3)
    optim.adamw_step([], [], [], [], step=1, lr=1e-3)
    assert optim.quantized_size(0) == (0, 0) and optim.quantized_size(1) == (128, 1) and optim.quantized_size(129) == (256, 2)


def test_preference_loss_object():
    loss = losses.get('preference_loss', beta=0.3, kind='hinge', length_normalized=True)
    assert isinstance(loss, losses.PreferenceLoss) and losses.RankingLossKey.PREFERENCE_LOSS in losses.RankingLossKey.all_keys()
    again = losses.PreferenceLoss.from_config(loss.get_config())
    assert again.get_config() == loss.get_config() == dict(reduction='auto', name=None, beta=0.3, kind='hinge', label_smoothing=0.0,
                                                           length_normalized=True)
    for kw in (dict(beta=0.0), dict(beta=float('nan')), dict(kind='other'), dict(label_smoothing=0.5), dict(reduction='mean'),
               dict(label_smoothing=0.1, kind='hinge')):
        with pytest.raises(ValueError):
            losses.PreferenceLoss(**kw)


def test_embedding_layer_and_builder():
    for bad in (dict(num_embeddings=0, embedding_dim=4), dict(num_embeddings=4, embedding_dim=0), dict(num_embeddings=4, embedding_dim=4, combiner='max')):
        with pytest.raises(ValueError):
            layers.Embedding(**bad)
    e = layers.Embedding(10, 4)
    assert e.weight.shape == (10, 4) and e.get_config() == dict(num_embeddings=10, embedding_dim=4, combiner='mean', scale=1.0)
    spec = {'ids': ra.data.FixedLenFeature([5], torch.int64, -1), 'x': ra.data.FixedLenFeature([3], torch.float32, 0.0)}
    b = pipeline.SimpleModelBuilder({}, spec, 'mask', embeddings={'ids': dict(num_embeddings=10, embedding_dim=4)}, hidden_layer_dims=[8])
    assert b._input_dim == 3 + 4 and isinstance(b.build().scorer, model.DNNScorer)
    b = pipeline.SimpleModelBuilder({}, spec, 'mask', embeddings={'ids': dict(num_embeddings=10, embedding_dim=4, combiner=None)},
                                    hidden_layer_dims=[8])
    assert b._input_dim == 3 + 20
    with pytest.raises(ValueError):
        pipeline.SimpleModelBuilder({}, spec, 'mask', embeddings={'other': dict(num_embeddings=10, embedding_dim=4)})
    assert {'adamw', 'adamw_8bit'} <= set(pipeline._OPTIMIZERS)


# ---------------------------------------------------------------- the plain forms themselves
def test_plain_embedding_gradient_against_torch():
    g = torch.Generator().manual_seed(1)
    table = torch.randn(7, 3, generator=g, dtype=torch.float64, requires_grad=True)
    ids = torch.tensor([[0, 3, -1], [3, 3, 6], [-1, -1, -1]])
    for combiner in (None, 'sum', 'mean'):
        rows = torch.nn.functional.embedding(ids.clamp(min=0), table) * (ids >= 0).unsqueeze(-1) * 2.0
        if combiner:
            rows = rows.sum(1)
            if combiner == 'mean':
                rows = rows / (ids >= 0).sum(1, keepdim=True).clamp(min=1)
        out, _ = T.embedding(table.detach(), ids, 2.0, combiner)
        assert torch.allclose(out, rows.detach(), atol=1e-12)
        up = torch.randn(rows.shape, generator=g, dtype=torch.float64)
        (want,) = torch.autograd.grad(rows, table, up)
        got, _, count = T.embedding_gradient(up, ids, 7, 2.0, combiner)
        assert torch.allclose(got, want, atol=1e-12) and count.tolist() == [1, 0, 0, 3, 0, 0, 1]


def test_plain_log_probs_gradient_against_differences():
    g = torch.Generator().manual_seed(2)
    x = torch.randn(4, 6, generator=g, dtype=torch.float64)
    t, up = torch.tensor([0, 5, -1, 2]), torch.randn(4, generator=g, dtype=torch.float64)
    got, _ = T.log_probs_gradient(up, x, t, 0.7)
    h = 1e-6
    for n in range(4):
        for v in range(6):
            hi, lo = x.clone(), x.clone()
            hi[n, v] += h
            lo[n, v] -= h
            diff = ((T.log_probs(hi, t, 0.7) - T.log_probs(lo, t, 0.7)) * up).sum() / (2 * h)
            assert abs(diff - got[n, v]) < 1e-8


@pytest.mark.parametrize('kind,smoothing', [('logistic', 0.0), ('logistic', 0.1), ('hinge', 0.0), ('squared', 0.0)])
@pytest.mark.parametrize('normalize', [False, True])
def test_plain_preference_gradient_against_differences(kind, smoothing, normalize):
    g = torch.Generator().manual_seed(3)
    y = torch.tensor([[2.0, 1.0, 0.0, 1.0], [1.0, 1.0, -1.0, 1.0], [3.0, -1.0, 0.0, 0.0]])
    lp, ref = torch.randn(3, 4, 5, generator=g, dtype=torch.float64), torch.randn(3, 4, 5, generator=g, dtype=torch.float64)
    mask = torch.rand(3, 4, 5, generator=g) < 0.6
    mask[0, 1] = False
    w = torch.tensor([1.0, 2.0, 0.5])
    args = (ref, mask, w, kind, 0.4, smoothing, normalize)
    loss, grad, _ = T.preference(y, lp, *args)
    assert loss[1] == 0 and not grad[1].any() and not grad[2, 1].any()
    h = 1e-6
    for at in [(0, 0, 0), (0, 2, 3), (0, 3, 1), (2, 0, 2), (2, 3, 4), (1, 0, 0)]:
        hi, lo = lp.clone(), lp.clone()
        hi[at] += h
        lo[at] -= h
        diff = (T.preference(y, hi, *args)[0] - T.preference(y, lo, *args)[0]).sum() / (2 * h)
        assert abs(diff - grad[at]) < 1e-7


def test_plain_adamw_against_torch():
    g = torch.Generator().manual_seed(4)
    p = torch.randn(50, generator=g, dtype=torch.float64)
    mine, m, v = p.clone(), torch.zeros(50, dtype=torch.float64), torch.zeros(50, dtype=torch.float64)
    theirs = torch.nn.Parameter(p.clone())
    opt = torch.optim.AdamW([theirs], lr=0.01, betas=(0.8, 0.99), eps=1e-8, weight_decay=0.1)
    for step in range(1, 6):
        grad = torch.randn(50, generator=g, dtype=torch.float64)
        theirs.grad = grad
        opt.step()
        mine, m, v, *_ = T.adamw(mine, grad, m, v, step, 0.01, (0.8, 0.99), 1e-8, 0.1)
        assert torch.allclose(mine, theirs.detach(), rtol=1e-12, atol=1e-14)


# ---------------------------------------------------------------- the optimizer's state
def held_state(p, step, bits=32):
    """The state of a parameter that took `step` steps, on the parameter's device (init_state() makes it on a GPU only)."""
    if bits == 32:
        return {'exp_avg': torch.full(p.shape, 0.5), 'exp_avg_sq': torch.full(p.shape, 0.25), 'step': step}
    codes, blocks = optim.quantized_size(p.numel())
    return {'exp_avg': torch.full((codes,), 3, dtype=torch.int8), 'exp_avg_sq': torch.full((codes,), 5, dtype=torch.uint8),
            'exp_avg_scale': torch.full((blocks,), 0.5), 'exp_avg_sq_scale': torch.full((blocks,), 0.25), 'step': step}


def test_a_refused_step_is_not_counted(monkeypatch):
    """A step that raises before it is launched (tensors that are refused, a capture that would freeze the count) leaves the
    counts: the next step's corrections are those of the steps that were taken."""
    p = torch.nn.Parameter(torch.zeros(3))
    opt = optim.AdamW([p])
    opt.state[p] = held_state(p, 2)
    p.grad = torch.ones(3)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    with pytest.raises(_lib.TfrHipError):                                   # not on a GPU
        opt.step()
    assert opt.state[p]['step'] == 2
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: True)
    with pytest.raises(RuntimeError, match='capturable'):
        opt.step()
    assert opt.state[p]['step'] == 2


def test_counted_adamw_arguments_are_checked_before_any_launch():
    lib = _lib.load()
    ptr, size = (ctypes.c_void_p * 1)(256), (ctypes.c_int64 * 1)(4)

    def call(steps=ptr, n=size, now=one, b1=0.9, count=1, dtype=0):
        return lib.tfr_adamw_counted(dtype, count, ptr, ptr, ptr, ptr, n, steps, None, None, 1e-3, b1, 0.999, 1e-8, 0.0, now, None)

    def call8(steps=ptr, n=size, now=one, scales=ptr, m=ptr):
        return lib.tfr_adamw8_counted(0, 1, ptr, ptr, m, scales, ptr, ptr, n, steps, None, None, 1e-3, 0.9, 0.999, 1e-8, 0.0, now, None)
    for f in (call, call8):
        assert f(steps=None) == -1 and f(steps=(ctypes.c_void_p * 1)(None)) == -1 and f(now=None) == -1
        assert f(n=(ctypes.c_int64 * 1)(-1)) == -1 and f(n=(ctypes.c_int64 * 1)(1 << 40)) == -1
    assert call(b1=1.0) == -1 and call(count=0) == -1 and call(count=89) == -1 and call(dtype=3) == -1
    assert call8(scales=None) == -1 and call8(m=(ctypes.c_void_p * 1)(260)) == -1


def same_places(before, s):
    return all(s[k] is t for k, t in before.items() if torch.is_tensor(t))


@pytest.mark.parametrize('bits', [32, 8])
def test_loading_fills_what_a_captured_step_holds(bits):
    """A captured step reads and writes the tensors that were there: a learning rate on the device, counts and moments keep their
    places, whatever the loaded state holds of them."""
    import copy
    ps = [torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(200))]
    lr = torch.tensor(0.25)
    opt = optim.AdamW(ps, lr=lr, capturable=True, state_bits=bits)
    fresh = copy.deepcopy(opt.state_dict())                                 # before any step: no moments, no counts
    for k, p in enumerate(ps):
        opt.state[p] = held_state(p, torch.tensor([4 + k]), bits)
    opt.param_groups[0]['step_count'] = torch.tensor([5])
    count, held = opt.param_groups[0]['step_count'], [dict(opt.state[p]) for p in ps]
    saved = copy.deepcopy(opt.state_dict())
    lr.fill_(0.5)
    count.fill_(9)
    for s in held:
        for t in s.values():
            t.zero_()

    def check(rate, counts, all_steps, moment):
        g = opt.param_groups[0]
        assert g['lr'] is lr and lr.item() == pytest.approx(rate) and g['step_count'] is count and count.item() == all_steps
        for p, s, n in zip(ps, held, counts):
            assert same_places(s, opt.state[p]) and set(s) == set(opt.state[p])
            assert s['step'].item() == n and s['exp_avg'].float().eq(moment).all()
    opt.load_state_dict(saved)
    check(0.25, (4, 5), 5, 0.5 if bits == 32 else 3)
    other = copy.deepcopy(saved)
    other['param_groups'][0]['lr'] = 0.125                                  # saved where the rate was a number
    opt.load_state_dict(other)
    check(0.125, (4, 5), 5, 0.5 if bits == 32 else 3)
    opt.load_state_dict(fresh)                                              # as at the start: nothing but zeros, in place
    check(0.25, (0, 0), 0, 0)
    partly = copy.deepcopy(saved)
    del partly['state'][1]
    opt.load_state_dict(partly)
    assert [s['step'].item() for s in held] == [4, 0] and not held[1]['exp_avg'].any() and held[0]['exp_avg'].any()
    assert all(same_places(s, opt.state[p]) for s, p in zip(held, ps))


def test_a_state_that_does_not_fit_changes_nothing():
    import copy
    ps = [torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(200))]
    opt = optim.AdamW(ps, lr=0.1)
    for k, p in enumerate(ps):
        opt.state[p] = held_state(p, 4 + k)
    bad = copy.deepcopy(opt.state_dict())
    bad['state'][0]['exp_avg'] = torch.ones(3)
    bad['state'][1]['exp_avg'] = torch.ones(199)
    bad['param_groups'][0]['lr'] = 7.0
    with pytest.raises(ValueError):
        opt.load_state_dict(bad)
    assert opt.param_groups[0]['lr'] == 0.1 and opt.state[ps[0]]['exp_avg'].eq(0.5).all() and opt.state[ps[1]]['step'] == 5


def test_a_learning_rate_on_the_device_follows_its_parameters():
    """Loaded into an optimizer whose rate is a number, a rate that was saved as a tensor is no part of the saved dict."""
    p, q = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3))
    lr = torch.tensor(0.25)
    saved = optim.AdamW([p], lr=lr, capturable=True).state_dict()
    opt = optim.AdamW([q], lr=0.5, capturable=True)
    opt.load_state_dict(saved)
    got = opt.param_groups[0]['lr']
    assert torch.is_tensor(got) and got is not lr and got.item() == 0.25 and got.device == q.device


def test_embedding_config_keeps_the_type():
    import json
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        e = layers.Embedding(10, 4, combiner='sum', scale=2.0, dtype=dtype)
        again = layers.Embedding(**json.loads(json.dumps(e.get_config())))
        assert again.weight.dtype == dtype and again.get_config() == e.get_config()
        assert layers.Embedding(10, 4).to(dtype).get_config() == layers.Embedding(10, 4, dtype=dtype).get_config()
    for bad in ('other', 'nn', None, 2):
        with pytest.raises(ValueError):
            layers.Embedding(10, 4, dtype=bad)


def test_a_state_without_moments_is_no_state(monkeypatch):
    """What a step that was refused leaves of a new parameter is saved and loaded as nothing."""
    import copy
    p, q = torch.nn.Parameter(torch.zeros(3)), torch.nn.Parameter(torch.zeros(3))
    opt, again = optim.AdamW([p]), optim.AdamW([q])
    p.grad = torch.ones(3)
    monkeypatch.setattr(torch.cuda, 'is_current_stream_capturing', lambda: False)
    with pytest.raises(_lib.TfrHipError):
        opt.step()
    again.state[q] = held_state(q, 4)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert again.state[q]['step'] == 0 and not again.state[q]['exp_avg'].any()


def test_loading_follows_parameters_that_moved():
    """State that is on another device than its parameter is replaced, not filled."""
    import copy
    p = torch.nn.Parameter(torch.zeros(3))
    opt = optim.AdamW([p], capturable=True)
    opt.state[p], opt.param_groups[0]['step_count'] = held_state(p, torch.tensor([4])), torch.tensor([4])
    saved = copy.deepcopy(opt.state_dict())
    opt.state[p] = {k: t.to('meta') for k, t in opt.state[p].items()}
    opt.param_groups[0]['step_count'] = opt.param_groups[0]['step_count'].to('meta')
    opt.load_state_dict(saved)
    assert all(t.device == p.device for t in opt.state[p].values()) and opt.state[p]['step'].item() == 4
    assert opt.param_groups[0]['step_count'].item() == 4 and opt.state[p]['exp_avg'].eq(0.5).all()
