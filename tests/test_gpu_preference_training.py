"""The training operators together, as a preference-tuned model uses them: token ids -> embedding -> scores over the vocabulary ->
token log probabilities of answers -> preference loss -> gradients -> AdamW, against the same step in float64 torch; and the
training pipeline with embedded id features and the AdamW optimizers."""
import pytest
import torch

pytestmark = pytest.mark.gpu
DEV = 'cuda'


def batch(vocab, B, L, tokens, seed):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, vocab, (B, L, tokens + 1), generator=g)
    length = torch.randint(1, tokens + 1, (B, L, 1), generator=g)
    mask = torch.arange(tokens) < length
    targets = torch.where(mask, ids[:, :, 1:], -1)
    inputs = torch.where(mask, ids[:, :, :-1], -1)
    return inputs, targets, mask, torch.randint(-1, 3, (B, L), generator=g).float()


def plain_step(table, weight, reference, inputs, targets, mask, y):
    """Loss and gradients in float64 on the CPU: log p(next | token) from a table, a product and a softmax."""
    table, weight = table.double().cpu().requires_grad_(), weight.double().cpu().requires_grad_()
    hidden = table[inputs.clamp(min=0)] * 4.0 * (inputs >= 0).unsqueeze(-1)
    logp = torch.log_softmax(hidden @ weight.t(), -1).gather(-1, targets.clamp(min=0).unsqueeze(-1)).squeeze(-1)
    ratio = torch.where(mask, logp - reference.double().cpu(), 0.0).sum(-1) * 0.5
    total = 0.0
    for n in range(y.shape[0]):
        pairs = [(i, j) for i in range(y.shape[1]) for j in range(y.shape[1]) if y[n, i] > y[n, j] >= 0]
        for i, j in pairs:
            total = total + torch.nn.functional.softplus(ratio[n, j] - ratio[n, i]) / len(pairs) / y.shape[0]
    grads = torch.autograd.grad(total, [table, weight])
    return total.detach(), grads


@pytest.mark.parametrize('autograd', [True, False])
def test_training_step(autograd):
    from ranking_amd import optim, preference
    from ranking_amd.embedding import embedding_grad, embedding_lookup
    from ranking_amd.keras.losses import PreferenceLoss
    vocab, dim, B, L, tokens = 211, 32, 6, 3, 19
    g = torch.Generator().manual_seed(1)
    start = [torch.randn(vocab, dim, generator=g) * 0.2, torch.randn(vocab, dim, generator=g) * 0.2]
    params = [torch.nn.Parameter(t.to(DEV)) for t in start]
    opt = optim.AdamW(params, lr=0.02, weight_decay=0.01)
    mirror = [torch.nn.Parameter(t.double()) for t in start]
    plain = torch.optim.AdamW(mirror, lr=0.02, weight_decay=0.01)
    loss_fn = PreferenceLoss(beta=0.5)
    for step in range(4):
        inputs, targets, mask, y = batch(vocab, B, L, tokens, step)
        on = [t.to(DEV) for t in (inputs, targets, mask, y)]
        table, weight = params
        with torch.no_grad():                                              # a reference model: where the training began
            ref = preference.token_log_probs((embedding_lookup(start[0].to(DEV), on[0], 4.0) @ start[1].to(DEV).t()), on[1])
        if autograd:
            opt.zero_grad()
            logits = embedding_lookup(table, on[0], 4.0) @ weight.t()
            loss = loss_fn(on[3], preference.token_log_probs(logits, on[1]), reference=ref, mask=on[2])
            loss.backward()
        else:
            with torch.no_grad():
                hidden = embedding_lookup(table, on[0], 4.0)
                logits = hidden @ weight.t()
                logp, stats = preference.token_log_probs_with_stats(logits, on[1])
                loss, dlogp = loss_fn.loss_and_grad(on[3], logp, reference=ref, mask=on[2])
                dlogits = preference.token_log_probs_grad(dlogp, logits, on[1], stats)
                weight.grad = dlogits.flatten(0, -2).t() @ hidden.flatten(0, -2)
                table.grad = embedding_grad(dlogits @ weight, on[0], vocab, 4.0)
        # float64 on the parameters as they are: sums of some 1e3 fp32 products, each 1e-7 of values up to 10
        want, grads = plain_step(table.detach(), weight.detach(), ref, inputs, targets, mask, y)
        assert abs(loss.item() - want.item()) < 1e-5
        for p, w in zip(params, grads):
            assert (p.grad.double().cpu() - w).norm() < 2e-5 * w.norm()
        for m, p in zip(mirror, params):                                   # the same gradients through torch's optimizer
            m.grad = p.grad.double().cpu()
        opt.step()
        plain.step()
        for m, p in zip(mirror, params):
            assert (p.double().cpu() - m).abs().max() < (step + 1) * 1e-6
    assert not params[0].grad[torch.tensor([v for v in range(vocab) if v not in set(inputs.flatten().tolist())], device=DEV)].any()


def test_training_step_in_a_graph():
    """The whole step without autograd, captured once and replayed on new batches = the eager step."""
    from ranking_amd import optim, preference
    from ranking_amd.embedding import embedding_grad, embedding_lookup
    from ranking_amd.keras.losses import PreferenceLoss
    vocab, dim = 97, 16
    loss_fn = PreferenceLoss(beta=0.5)
    results = []
    for captured in (False, True):
        g = torch.Generator().manual_seed(1)
        table, weight = (torch.nn.Parameter((torch.randn(vocab, dim, generator=g) * 0.2).to(DEV)) for _ in range(2))
        table.grad, weight.grad = torch.zeros_like(table), torch.zeros_like(weight)
        opt = optim.AdamW([table, weight], lr=0.02, capturable=True, state_bits=8)
        opt.init_state()
        held = [t.to(DEV) for t in batch(vocab, 4, 2, 11, 0)]

        @torch.no_grad()
        def step():
            hidden = embedding_lookup(table, held[0], 4.0)
            logits = hidden @ weight.t()
            logp, stats = preference.token_log_probs_with_stats(logits, held[1])
            loss, dlogp = loss_fn.loss_and_grad(held[3], logp, mask=held[2])
            dlogits = preference.token_log_probs_grad(dlogp, logits, held[1], stats)
            weight.grad.copy_(dlogits.flatten(0, -2).t() @ hidden.flatten(0, -2))
            table.grad.copy_(embedding_grad(dlogits @ weight, held[0], vocab, 4.0))
            opt.step()
            return loss
        if captured:
            saved = [t.detach().clone() for t in (table, weight)]
            state = __import__('copy').deepcopy(opt.state_dict())
            s = torch.cuda.Stream()
            s.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(s):
                step()
            torch.cuda.current_stream().wait_stream(s)
            opt.load_state_dict(state)
            with torch.no_grad():
                table.copy_(saved[0])
                weight.copy_(saved[1])
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                out = step()
        losses = []
        for k in range(10):                                                # 0, 1 and 3 hold no pair: those steps only decay
            for h, t in zip(held, batch(vocab, 4, 2, 11, k)):
                h.copy_(t)
            if captured:
                graph.replay()
            else:
                out = step()
            torch.cuda.synchronize()
            losses.append(out.item())
        results.append((losses, table.detach().clone(), weight.detach().clone()))
    assert results[0][0] == results[1][0]
    assert torch.equal(results[0][1], results[1][1]) and torch.equal(results[0][2], results[1][2])


def test_autograd_in_a_graph():
    """Forward and autograd.grad captured together (every graph before it is gone), replayed on new batches = eager."""
    from ranking_amd import preference
    from ranking_amd.embedding import embedding_lookup
    from ranking_amd.keras.losses import PreferenceLoss
    vocab, dim = 97, 16
    g = torch.Generator().manual_seed(3)
    table, weight = ((torch.randn(vocab, dim, generator=g) * 0.2).to(DEV).requires_grad_() for _ in range(2))
    loss_fn = PreferenceLoss(beta=0.5)
    held = [t.to(DEV) for t in batch(vocab, 4, 2, 11, 0)]

    def step():
        logits = embedding_lookup(table, held[0], 4.0) @ weight.t()
        loss = loss_fn(held[3], preference.token_log_probs(logits, held[1]), mask=held[2])
        return [loss.detach(), *torch.autograd.grad(loss, [table, weight])]
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        step()
    torch.cuda.current_stream().wait_stream(s)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    pairs = 0
    for k in range(10):
        new = batch(vocab, 4, 2, 11, k)
        for h, t in zip(held, new):
            h.copy_(t)
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        y = new[3]
        has = bool(((y[:, 0] != y[:, 1]) & (y >= 0).all(1)).any())          # without a pair the loss is 0 and so are its gradients
        assert all(torch.equal(a, b) for a, b in zip(out, want)) and bool(want[1].any()) == bool(want[2].any()) == has
        pairs += has
    assert pairs >= 3


def work_of(seed, dtype):
    """One of two programs that run at the same time: its inputs, and a call that gives the outputs of every operator on them."""
    from ranking_amd import optim, preference
    from ranking_amd.embedding import embedding_grad, embedding_lookup
    from ranking_amd.keras.losses import PreferenceLoss
    g = torch.Generator().manual_seed(seed)
    vocab, dim, n = 5000 + seed, 40, 9000
    table = torch.randn(vocab, dim, generator=g).to(dtype).to(DEV)
    ids = torch.randint(-1, vocab, (n,), generator=g).to(DEV)
    bags = torch.randint(-1, vocab, (600, 7), generator=g).to(DEV)
    logits = torch.randn(6, 40000, generator=g).to(dtype).to(DEV)
    targets = torch.randint(-1, 40000, (6,), generator=g).to(DEV)
    up, loss = torch.randn(6, generator=g).to(DEV), PreferenceLoss(beta=0.5)
    lp = (-torch.rand(3, 2, 6000, generator=g)).to(DEV)
    y = torch.tensor([[1.0, 0.0]] * 3, device=DEV)

    def run():
        rows = embedding_lookup(table, ids, 2.0)
        means = embedding_lookup(table, bags, combiner='mean')
        logp, stats = preference.token_log_probs_with_stats(logits, targets)
        param, m, v = table.clone(), torch.zeros(table.shape, device=DEV), torch.zeros(table.shape, device=DEV)
        grad = embedding_grad(rows, ids, vocab, 2.0)
        optim.adamw_step([param], [grad], [m], [v], step=1, lr=0.1)
        codes, blocks = optim.quantized_size(param.numel())
        m8 = torch.zeros(codes, dtype=torch.int8, device=DEV), torch.zeros(blocks, device=DEV)
        v8 = torch.zeros(codes, dtype=torch.uint8, device=DEV), torch.zeros(blocks, device=DEV)
        optim.adamw_step([param], [grad], [m8], [v8], step=1, lr=0.1)
        return [rows, means, grad, embedding_grad(means, bags, vocab, combiner='mean'), logp,
                preference.token_log_probs_grad(up, logits, targets, stats), *loss.loss_and_grad(y, lp), param, m, v, *m8, *v8]
    return run


@pytest.mark.parametrize('threads', [False, True])
def test_two_programs_at_once(threads):
    """Two streams, driven by one thread or by one each, run every operator on inputs of their own: the same bits as alone."""
    import threading
    work = [work_of(1, torch.float32), work_of(2, torch.bfloat16)]
    want = [run() for run in work]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in work], [[], []]

    def drive(k):
        with torch.cuda.stream(streams[k]):
            got[k].append(work[k]())
    if threads:
        def many(k):
            for _ in range(5):
                drive(k)
        both = [threading.Thread(target=many, args=(k,)) for k in range(2)]
        for t in both:
            t.start()
        for t in both:
            t.join()
    else:
        for _ in range(5):
            drive(0)
            drive(1)
    torch.cuda.synchronize()
    for k in range(2):
        assert len(got[k]) == 5
        for outs in got[k]:
            assert all(torch.equal(a, b) for a, b in zip(outs, want[k]))


@pytest.mark.parametrize('optimizer', ['adamw', 'adamw_8bit'])
@pytest.mark.parametrize('loss', ['softmax_loss', 'preference_loss'])
def test_pipeline_with_embedded_features(tmp_path, optimizer, loss):
    import ranking_amd as ra
    pl = ra.keras.pipeline
    g = torch.Generator().manual_seed(2)

    def dataset():
        while True:
            ids = torch.randint(-1, 40, (8, 10, 6), generator=g)
            yield {'tokens': ids.float(), 'x': torch.randn(8, 10, 3, generator=g), 'mask': torch.ones(8, 10, dtype=torch.bool)}, torch.randint(0, 3, (8, 10), generator=g).float()
    spec = {'tokens': ra.data.FixedLenFeature([6], torch.float32, -1.0), 'x': ra.data.FixedLenFeature([3], torch.float32, 0.0)}
    hp = pl.PipelineHparams(model_dir=str(tmp_path), num_epochs=1, steps_per_epoch=3, validation_steps=1, learning_rate=0.01, loss=loss, optimizer=optimizer)
    builder = pl.SimpleModelBuilder({}, spec, 'mask', embeddings={'tokens': dict(num_embeddings=40, embedding_dim=5)}, hidden_layer_dims=[16], dropout=0.0)
    pipe = pl.SimplePipeline(builder, pl.NullDatasetBuilder(dataset(), dataset()), hp)
    history = pipe.train_and_validate()
    assert torch.isfinite(torch.tensor(history['loss'] + history['val_loss'])).all()
    table = pipe.model.scorer._embeddings['tokens'].weight
    assert table.grad is not None and table.grad.abs().sum() > 0 and torch.isfinite(table).all()


def test_forward_mode_is_refused():
    """None of the operators has a forward-mode derivative: a tensor that carries a tangent is refused, with and without gradients
    (the call used to give a result without one)."""
    import torch.autograd.forward_ad as fwAD
    from ranking_amd import preference
    from ranking_amd.embedding import embedding_lookup
    from ranking_amd.keras.losses import PreferenceLoss
    x, ids, y = torch.randn(6, 8, device=DEV), torch.tensor([1, 5, -1], device=DEV), torch.ones(6, 8, device=DEV)
    calls = (lambda t: embedding_lookup(t, ids), lambda t: embedding_lookup(t, ids.view(1, 3), combiner='mean'),
             lambda t: preference.token_log_probs(t[:3], ids), lambda t: PreferenceLoss()(y, t))
    plain = [call(x) for call in calls]
    with fwAD.dual_level():
        assert all(torch.equal(call(x), want) for call, want in zip(calls, plain))      # a level alone changes nothing
        dual = fwAD.make_dual(x, torch.ones_like(x))
        for call in calls:
            for grad in (True, False):
                with torch.set_grad_enabled(grad), pytest.raises(NotImplementedError):
                    call(dual)
    for call in calls[:3]:
        with pytest.raises((NotImplementedError, RuntimeError)):
            torch.func.jvp(call, (x,), (torch.ones_like(x),))
