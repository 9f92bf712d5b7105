"""AdamW with 32-bit and 8-bit moments (csrc/adamw.hip, ranking_amd.optim) on the GPU against the plain 64-bit form; the bounds
are derived in tests/training_ops.py (adamw).  8-bit codes are the nearest to fp64 values: equal but next to a border."""
import math

import pytest
import torch

from tests import training_ops as T

pytestmark = pytest.mark.gpu
DEV = 'cuda'
DTYPES = [torch.float32, torch.bfloat16, torch.float16]
HYPER = dict(lr=0.01, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.1)


def O():
    from ranking_amd import optim
    return optim


def make(sizes, dtype, seed=0):
    g = torch.Generator().manual_seed(seed + len(sizes))
    rnd = lambda n, s: torch.randn(n, generator=g) * s                      # noqa: E731
    return ([rnd(n, 1.0).to(dtype) for n in sizes], [rnd(n, 0.1).to(dtype) for n in sizes], [rnd(n, 0.05) for n in sizes],
            [rnd(n, 0.1) ** 2 for n in sizes])


def on(ts):
    return [t.to(DEV) for t in ts]


def check32(p, g, m, v, step=7, **hyper):
    h = dict(HYPER, **hyper)
    P, G, M, V = on(p), on(g), on(m), on(v)
    O().adamw_step(P, G, M, V, step=step, **h)
    for k in range(len(p)):
        p1, m1, v1, dm, dv, dp = T.adamw(p[k], g[k], m[k], v[k], step, h['lr'], h['betas'], h['eps'], h['weight_decay'])
        T.assert_within(M[k], m1, dm, 'exp_avg %d' % k)
        T.assert_within(V[k], v1, dv, 'exp_avg_sq %d' % k)
        T.assert_within(P[k], p1, dp + T.half(p[k].dtype) * (p1.abs() + dp) + T.tiny(p[k].dtype), 'param %d' % k)
    return P, M, V


SIZES = [[1], [5, 0, 4096], [4095, 4097, 3], [100003], [17] * 200]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('sizes', SIZES, ids=str)
def test_32_bits(dtype, sizes):
    check32(*make(sizes, dtype))


@pytest.mark.parametrize('hyper', [dict(weight_decay=0.0), dict(betas=(0.0, 0.0)), dict(eps=1.0), dict(lr=0.0), dict(betas=(0.8, 0.95), step=1),
                                   dict(step=1000000)], ids=str)
def test_hyperparameters(hyper):
    args = make([777], torch.float32)
    check32(*args, **hyper)
    check8(*args[:2], **hyper)


def quantized(p, seed=3):
    """Random codes and scales for parameters p: (codes m, scales m, codes v, scales v) a tensor."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for t in p:
        n, blocks = O().quantized_size(t.numel())
        cm, cv = torch.randint(-127, 128, (n,), generator=g), torch.randint(0, 256, (n,), generator=g)
        cm[t.numel():], cv[t.numel():] = 0, 0
        cm[:t.numel()][cv[:t.numel()] == 0] = 0
        out.append((cm.to(torch.int8), torch.rand(blocks, generator=g) * 1e-3, cv.to(torch.uint8), torch.rand(blocks, generator=g) * 1e-3))
    return out


def wide(codes, scales, n):
    return (codes.double() * scales.double().repeat_interleave(128))[:n]


def check8(p, g, state=None, step=7, **hyper):
    h = dict(HYPER, **hyper)
    state = quantized(p) if state is None else state
    P, G = on(p), on(g)
    S = [tuple(x.to(DEV) for x in s) for s in state]
    O().adamw_step(P, G, [(s[0], s[1]) for s in S], [(s[2], s[3]) for s in S], step=step, **h)
    for k, (cm, sm, cv, sv) in enumerate(state):
        n = p[k].numel()
        m, v = wide(cm, sm, n), wide(cv, sv, n) ** 2
        p1, m1, v1, dm, dv, dp = T.adamw(p[k], g[k], m, v, step, h['lr'], h['betas'], h['eps'], h['weight_decay'])
        cm1, cv1, sm1, sv1, sure_m, sure_v = T.adamw_codes(m1, v1)
        got = [x.cpu() for x in S[k]]
        # scales are rounded once, from fp64
        assert torch.equal(got[1], sm1) and torch.equal(got[3], sv1), 'scales of %d' % k
        off_m, off_v = (got[0].double() - cm1).abs(), (got[2].double() - cv1).abs()
        assert off_m.numel() == 0 or (off_m.max() <= 1 and not off_m[sure_m].any()), 'codes of exp_avg %d' % k
        assert off_v.numel() == 0 or (off_v.max() <= 1 and not off_v[sure_v].any()), 'codes of exp_avg_sq %d' % k
        T.assert_within(P[k], p1, dp + T.half(p[k].dtype) * (p1.abs() + dp) + T.tiny(p[k].dtype), 'param %d' % k)
        assert not got[0][n:].any() and not got[2][n:].any()
        T.assert_within(O().dequantize_exp_avg(S[k][0], S[k][1]), wide(got[0], got[1], cm.numel()), T.U * wide(got[0], got[1], cm.numel()).abs() + 1e-45)
        root = wide(got[2], got[3], cm.numel())
        T.assert_within(O().dequantize_exp_avg_sq(S[k][2], S[k][3]), root ** 2, 3.1 * T.U * root ** 2 + 1e-45)
    return P, S


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('sizes', [[1], [127, 128, 129, 0], [2047, 2048, 2049, 4097], [100003], [17] * 130], ids=str)
def test_8_bits(dtype, sizes):
    check8(*make(sizes, dtype)[:2])


def test_8_bits_from_zero():
    """The first step: all codes zero, scales zero; a block without a gradient stays zero, small roots keep a code of 1."""
    n = 400
    g = torch.randn(n, generator=torch.Generator().manual_seed(5))
    g[128:256] = 0.0
    g[300] = 1e-6
    zero = [(torch.zeros(512, dtype=torch.int8), torch.zeros(4), torch.zeros(512, dtype=torch.uint8), torch.zeros(4))]
    _, S = check8([torch.randn(n)], [g], zero, step=1)
    assert not S[0][0][128:256].any() and not S[0][2][128:256].any() and S[0][2][300] == 1
    assert S[0][1][1] == 0 and S[0][3][1] == 0


def test_8_bits_of_tiny_and_huge_gradients():
    g = torch.tensor([1e-30, -1e-38, 1e-42, 0.0] * 40 + [1e18, -1e15, 1.0, 0.0] * 40)
    zero = [(torch.zeros(384, dtype=torch.int8), torch.zeros(3), torch.zeros(384, dtype=torch.uint8), torch.zeros(3))]
    P, S = check8([torch.ones(320)], [g], zero, step=1)
    assert torch.isfinite(P[0]).all()


def test_8_bits_keep_a_lost_element_to_itself():
    """NaN and infinite gradients poison their own element for good, and nothing else of their block."""
    p, g = torch.ones(256), torch.randn(256, generator=torch.Generator().manual_seed(6))
    bad, good = g.clone(), g.clone()
    bad[3], bad[40], good[3], good[40] = float('nan'), float('inf'), 0.0, 0.0
    state = quantized([p])
    _, S = check8([p], [good], [tuple(x.clone() for x in state[0])])
    P, B = on([p]), [tuple(x.to(DEV) for x in s) for s in state]
    O().adamw_step(P, on([bad]), [B[0][:2]], [B[0][2:]], step=7, **HYPER)
    assert P[0].isnan().nonzero().flatten().tolist() in ([3], [3, 40])
    assert B[0][0][3] == -128 and B[0][0][40] == -128 and O().dequantize_exp_avg(*B[0][:2]).isnan().sum() == 2
    rest = torch.ones(256, dtype=torch.bool)
    rest[[3, 40]] = False
    same = state[0][0][rest].abs().max() == state[0][0].abs().max()
    if same:
        assert torch.isfinite(B[0][1]).all() and torch.isfinite(B[0][3]).all()
    O().adamw_step(P, on([good]), [B[0][:2]], [B[0][2:]], step=8, **HYPER)
    assert P[0].isnan().nonzero().flatten().tolist() == [3, 40]


@pytest.mark.parametrize('dtype', DTYPES)
def test_shifted_and_shaped_tensors(dtype):
    """Views of a flat buffer at odd places, matrices, scalars."""
    p, g, m, v = make([5000], dtype)
    flat = [t[0].to(DEV) for t in (p, g, m, v)]
    cuts = [(1, 130), (133, 4097), (4235, 1), (4240, 64)]
    views = [[f[a:a + n] for a, n in cuts] for f in flat]
    O().adamw_step(*views, step=3, **HYPER)
    for k, (a, n) in enumerate(cuts):
        p1, m1, v1, dm, dv, dp = T.adamw(p[0][a:a + n], g[0][a:a + n], m[0][a:a + n], v[0][a:a + n], 3, 0.01, (0.9, 0.999), 1e-8, 0.1)
        T.assert_within(views[0][k], p1, dp + T.half(dtype) * (p1.abs() + dp) + T.tiny(dtype))
        T.assert_within(views[2][k], m1, dm)
    held = torch.ones(5000, dtype=torch.bool)
    for a, n in cuts:
        held[a:a + n] = False
    assert torch.equal(flat[0].cpu()[held], p[0][held]) and torch.equal(flat[2].cpu()[held], m[0][held])   # what lies between is left
    p, g = make([600], dtype)[:2]
    state = quantized([p[0][1:]])
    P = p[0].to(DEV)
    S = [tuple(x.to(DEV) for x in state[0])]
    O().adamw_step([P[1:]], [g[0].to(DEV)[1:]], [S[0][:2]], [S[0][2:]], step=2, **HYPER)
    Q, R = check8([p[0][1:].clone()], [g[0][1:].clone()], state, step=2)
    assert torch.equal(P[1:], Q[0]) and P[0] == p[0][0].to(DEV) and all(torch.equal(a, b) for a, b in zip(S[0], R[0]))


@pytest.mark.parametrize('bits,dtype', [(32, torch.float32), (32, torch.bfloat16), (8, torch.float32), (8, torch.bfloat16)])
def test_launches_beyond_the_caches(bits, dtype):
    """48 M elements, a launch that goes past the caches: the same bits as in parts that do not."""
    n = 48 * 1024 * 1024 + 77
    p, g = (torch.randn(n, device=DEV) * s for s in (1.0, 0.1))
    whole, parts = [p.to(dtype), g.to(dtype)], [p.to(dtype), g.to(dtype)]
    codes, blocks = O().quantized_size(n)
    for t in (whole, parts):
        t += ([torch.zeros(codes, dtype=torch.int8, device=DEV), torch.zeros(blocks, device=DEV), torch.zeros(codes, dtype=torch.uint8, device=DEV),
               torch.zeros(blocks, device=DEV)] if bits == 8 else [torch.zeros(n, device=DEV), torch.zeros(n, device=DEV)])

    def step(t, a, b, k):
        q = (a // 128, (b + 127) // 128)
        if bits == 8:
            moments = [(t[i][q[0] * 128:q[1] * 128], t[i + 1][q[0]:q[1]]) for i in (2, 4)]
        else:
            moments = [t[i][a:b] for i in (2, 3)]
        O().adamw_step([t[0][a:b]], [t[1][a:b]], [moments[0]], [moments[1]], step=k, **HYPER)
    cut = 4 * 1024 * 1024
    for k in (1, 2):
        step(whole, 0, n, k)
        for a in range(0, n, cut):
            step(parts, a, min(n, a + cut), k)
    assert all(torch.equal(x, y) for x, y in zip(whole, parts))


def test_mixed_types_in_one_call():
    a, b = make([100, 50], torch.float32), make([200], torch.bfloat16)
    mixed = [x + y for x, y in zip(a, b)]
    check32(*mixed)


def test_offsets_beyond_32_bits():
    n = (1 << 32) + 200
    p, g = torch.zeros(n, dtype=torch.bfloat16, device=DEV), torch.zeros(n, dtype=torch.bfloat16, device=DEV)
    codes, blocks = O().quantized_size(n)
    m, v = torch.zeros(codes, dtype=torch.int8, device=DEV), torch.zeros(codes, dtype=torch.uint8, device=DEV)
    sm, sv = torch.zeros(blocks, device=DEV), torch.zeros(blocks, device=DEV)
    p[-1], g[-1] = 1.0, 0.5
    O().adamw_step([p], [g], [(m, sm)], [(v, sv)], step=1, lr=0.5, weight_decay=0.0)
    assert p[-1] == 0.5 and m[n - 1] == 127 and v[n - 1] == 255 and not p[:-1].any() and not m[: n - 128].any()
    assert O().dequantize_exp_avg(m[-256:], sm[-2:])[n - codes - 1].item() == pytest.approx(0.05, rel=1e-6)


# ---------------------------------------------------------------- the optimizer object
def params(dtype=torch.float32, seed=0):
    g = torch.Generator().manual_seed(seed)
    return [torch.nn.Parameter((torch.randn(s, generator=g)).to(dtype).to(DEV)) for s in ((33, 7), (5,), (300,), ())]


def grads(ps, seed):
    g = torch.Generator().manual_seed(seed)
    for p in ps:
        p.grad = torch.randn(p.shape, generator=g).to(p.dtype).to(DEV)


def test_object_against_the_plain_form():
    """Ten steps; a parameter that gets no gradient for a while keeps its own count; a gradient of other strides."""
    ps = params()
    opt = O().AdamW(ps, **HYPER)
    plain = [(p.detach().double().cpu(), torch.zeros(p.shape, dtype=torch.float64), torch.zeros(p.shape, dtype=torch.float64), 0) for p in ps]
    for step in range(10):
        grads(ps, step)
        ps[0].grad = ps[0].grad.t().contiguous().t()
        if step in (2, 3):
            ps[2].grad = None
        for k, p in enumerate(ps):
            if p.grad is not None:
                q, m, v, t = plain[k]
                q, m, v, *_ = T.adamw(q, p.grad, m, v, t + 1, 0.01, (0.9, 0.999), 1e-8, 0.1)
                plain[k] = (q, m, v, t + 1)
        opt.step()
    for p, (q, m, v, t) in zip(ps, plain):
        # ten steps of at most lr / (1 - beta1) each, every one off by some 20 roundings
        assert torch.allclose(p.detach().double().cpu(), q, rtol=0, atol=10 * 20 * T.U * (q.abs().max() + 1).item())
        assert opt.state[p]['step'] == t
    assert opt.step(lambda: 3.0) == 3.0


@pytest.mark.parametrize('bits', [8, 32])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_state_dict_round_trip(bits, dtype):
    """Saved and loaded, the optimizer goes on bit for bit, and the moments keep their types."""
    ps = params(dtype)
    opt = O().AdamW(ps, state_bits=bits, **HYPER)
    for step in range(3):
        grads(ps, step)
        opt.step()
    import io
    buf = io.BytesIO()
    torch.save(opt.state_dict(), buf)
    buf.seek(0)
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    again = O().AdamW(qs, state_bits=bits, lr=1.0)
    again.load_state_dict(torch.load(buf, weights_only=True, map_location='cpu'))
    for step in range(3, 5):
        grads(ps, step)
        grads(qs, step)
        opt.step()
        again.step()
    for p, q in zip(ps, qs):
        assert torch.equal(p, q)
        assert {k: getattr(x, 'dtype', None) for k, x in opt.state[p].items()} == {k: getattr(x, 'dtype', None) for k, x in again.state[q].items()}
    with pytest.raises(ValueError):
        O().AdamW([torch.nn.Parameter(torch.zeros(3, device=DEV)) for _ in range(4)], state_bits=bits).load_state_dict(opt.state_dict())


@pytest.mark.parametrize('bits', [8, 32])
def test_captured_steps(bits):
    """A captured step that counts on the device, replayed with eager steps between and a learning rate that changes, is bit for
    bit the eager one that counts there too, and within rounding of the one that counts on the host."""
    runs = []
    for captured in (True, False):
        ps = params()
        lr = torch.tensor(0.01, device=DEV)
        opt = O().AdamW(ps, lr=lr, betas=(0.9, 0.999), weight_decay=0.1, state_bits=bits, capturable=True)
        held = [torch.zeros_like(p) for p in ps]
        for p, h in zip(ps, held):
            p.grad = h

        def new(step):
            g = torch.Generator().manual_seed(step)
            for h in held:
                h.copy_(torch.randn(h.shape, generator=g))
        graph = None
        if captured:
            opt.init_state()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
        for step in range(6):
            new(step)
            lr.fill_(0.01 / (1 + step))
            if captured and step != 3:
                graph.replay()
            else:
                opt.step()
            torch.cuda.synchronize()
        assert opt.param_groups[0]['step_count'].item() == 6
        runs.append(ps)
        if captured:                                                       # loading fills what the graph holds
            saved = opt.state_dict()
            before = [p.detach().clone() for p in ps]
            import copy
            saved = copy.deepcopy(saved)
            graph.replay()
            opt.load_state_dict(saved)
            assert opt.param_groups[0]['step_count'].item() == 6
            with torch.no_grad():
                for p, b in zip(ps, before):
                    p.copy_(b)
    for a, b in zip(*runs):
        assert torch.equal(a, b)
    ps = params()
    opt = O().AdamW(ps, lr=0.01, weight_decay=0.1, state_bits=bits)
    for step in range(6):
        g = torch.Generator().manual_seed(step)
        for p in ps:
            p.grad = torch.randn(p.shape, generator=g).to(DEV)
        opt.param_groups[0]['lr'] = torch.tensor(0.01 / (1 + step), dtype=torch.float32).item()
        opt.step()
    for a, b in zip(runs[0], ps):
        # the coefficients come from pow() of the host and of the device: a rounding a step
        assert torch.allclose(a, b, rtol=0, atol=6 * 20 * T.U * (b.abs().max() + 1).item())


def test_capture_needs_its_state():
    ps = params()
    grads(ps, 0)
    opt = O().AdamW(ps)
    opt.step()
    frozen = O().AdamW(ps, capturable=True)
    for o, what in ((opt, 'capturable'), (frozen, 'init_state')):
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with pytest.raises(RuntimeError, match=what):
            with torch.cuda.graph(graph):
                o.step()


def test_other_stream():
    args = make([5000, 30], torch.float32)
    want = check32(*args)
    P, G, M, V = (on(t) for t in args)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        O().adamw_step(P, G, M, V, step=7, **HYPER)
    torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for a, b in zip(P + M + V, want[0] + want[1] + want[2]))


def test_refusals():
    z = lambda n=4, d=torch.float32: torch.zeros(n, dtype=d, device=DEV)    # noqa: E731
    step = lambda *a, **k: O().adamw_step(*[[x] for x in a], **{**dict(step=1, lr=1e-3), **k})   # noqa: E731
    p = z()
    eight = ((z(128, torch.int8), z(1)), (z(128, torch.uint8), z(1)))
    for bad in (lambda: step(z(d=torch.float64), z(d=torch.float64), z(), z()), lambda: step(p, z(3), z(), z()), lambda: step(p, z(d=torch.bfloat16), z(), z()),
                lambda: step(p, z(), z(3), z()), lambda: step(p, z(), z(), z(d=torch.bfloat16)), lambda: step(z(8)[::2], z(), z(), z()),
                lambda: step(p, z(8)[::2], z(), z()), lambda: step(p, z(), eight[0], z()), lambda: step(p, z(), eight[1], eight[0]),
                lambda: step(p, z(), (z(4, torch.int8), z(1)), eight[1]), lambda: step(p, z(), z(), z(), lr=torch.tensor(1.0, device=DEV)),
                lambda: step(p, z(), (z(136, torch.int8)[4:132], z(1)), eight[1]),
                lambda: O().adamw_step([p, p], [z(), z()], [z(), z()], [z(), z()], step=1, lr=1e-3),
                lambda: step(p, z(), z(), z(), now=z(2)), lambda: step(p, z(), z(), z(), now=z(3, torch.float64)),
                lambda: step(p, z(), z(), z(), now=torch.zeros(3)),
                lambda: O().AdamW([dict(params=[torch.nn.Parameter(z())], state_bits=16)]),
                lambda: O().AdamW([torch.nn.Parameter(z())]).add_param_group(dict(params=[torch.nn.Parameter(z())], lr=-1.0)),
                lambda: O().dequantize_exp_avg(z(130, torch.int8), z(2)), lambda: O().dequantize_exp_avg(z(128, torch.uint8), z(1)),
                lambda: O().dequantize_exp_avg_sq(z(128, torch.uint8), z(2))):
        with pytest.raises(ValueError):
            bad()
    sparse = torch.nn.Parameter(torch.zeros(4, 2, device=DEV))
    sparse.grad = torch.sparse_coo_tensor(torch.tensor([[1]]), torch.ones(1, 2), (4, 2)).to(DEV)
    with pytest.raises(ValueError):
        O().AdamW([sparse]).step()
    assert math.isfinite(p.sum().item())


def test_stale_graphs_are_refused():
    """A step changes the parameters that an earlier graph saved: its backward raises instead of mixing old and new values."""
    w = torch.nn.Parameter(torch.ones(4, 4, device=DEV))
    x = torch.ones(2, 4, device=DEV, requires_grad=True)
    opt = O().AdamW([w], lr=0.1)
    loss = (x @ w).sum()
    loss.backward(retain_graph=True)
    opt.step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()
    with torch.inference_mode():                                           # tensors without a version are stepped all the same
        a, b = torch.ones(3, device=DEV), torch.zeros(3, device=DEV)
        O().adamw_step([a], [torch.ones_like(a)], [b], [torch.zeros_like(a)], step=1, lr=0.1, weight_decay=0.0)
        assert torch.allclose(a, torch.full_like(a, 0.9), atol=1e-6)


# ---------------------------------------------------------------- counts of a capturable group
@pytest.mark.parametrize('bits', [8, 32])
@pytest.mark.parametrize('replayed', [False, True])
def test_counts_on_the_device_are_a_parameters_own(bits, replayed):
    """A parameter that is frozen at first, or for a while, is corrected by the number of its own steps, as it is where the host
    counts: lr (m / (1 - beta1)) / sqrt(v / (1 - beta2)) = lr at its first step, not 3.2 lr.  `replayed`: the steps of all parameters
    are a graph that was captured before any was missed."""
    runs = []
    for capturable in (True, False):
        ps = params()
        held = [torch.zeros_like(p) for p in ps]
        opt = O().AdamW(ps, lr=0.01, weight_decay=0.1, state_bits=bits, capturable=capturable)
        graph = None
        if capturable and replayed:
            for p, h in zip(ps, held):
                p.grad = h
            opt.init_state()
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
        for step in range(12):
            g = torch.Generator().manual_seed(step)
            for h in held:
                h.copy_(torch.randn(h.shape, generator=g))
            missing = {2} if step < 6 else {0, 3} if step in (7, 8) else set()
            for k, (p, h) in enumerate(zip(ps, held)):
                p.grad = None if k in missing else h
            before = ps[2].detach().clone()
            if graph is not None and not missing:
                graph.replay()
            else:
                opt.step()
            if step == 6:                                      # the late one's first step: every element moves by lr, and decays
                moved = (ps[2] - before * (1 - 0.01 * 0.1)).abs()
                assert (moved - 0.01).abs().max() < 1e-4 * 0.01 + 4 * T.U * before.abs().max()
        torch.cuda.synchronize()
        assert [int(opt.state[p]['step']) for p in ps] == [10, 12, 6, 10]
        runs.append((ps, [opt.state[p] for p in ps]))
    for a, b in zip(runs[0][0], runs[1][0]):
        # the coefficients come from pow() of the host and of the device: a rounding a step
        assert torch.allclose(a, b, rtol=0, atol=12 * 20 * T.U * (b.abs().max() + 1).item())
    for a, b in zip(runs[0][1], runs[1][1]):
        for key in ('exp_avg', 'exp_avg_sq'):
            assert torch.equal(a[key], b[key])                 # the moments do not hang on the count


def test_counts_of_many_tensors_and_types():
    """More tensors than a launch holds, two types in a group, one empty: as where the host counts."""
    runs = []
    for capturable in (True, False):
        g = torch.Generator().manual_seed(1)
        ps = [torch.nn.Parameter(torch.randn(n % 13, generator=g).to(torch.bfloat16 if n % 3 == 0 else torch.float32).to(DEV)) for n in range(1, 200)]
        opt = O().AdamW(ps, lr=0.01, capturable=capturable)
        for step in range(3):
            for k, p in enumerate(ps):
                grad = torch.randn(p.shape, generator=g).to(p.dtype).to(DEV)
                p.grad = grad if (k + step) % 5 or step == 2 else None
            opt.step()
        runs.append((ps, [int(opt.state[p]['step']) for p in ps]))
    assert all(a == b for a, b, p in zip(runs[0][1], runs[1][1], runs[0][0]) if p.numel())
    for a, b in zip(runs[0][0], runs[1][0]):
        assert torch.allclose(a.float(), b.float(), rtol=0 if a.dtype == torch.float32 else 2 ** -8, atol=3 * 20 * T.U * 5)


@pytest.mark.parametrize('bits', [8, 32])
def test_counts_are_saved_and_loaded(bits):
    """A saved capturable state goes on bit for bit, with the counts of its parameters; one that holds the group's count alone gives
    it to each; and a group whose `capturable` is switched keeps its counts."""
    import copy
    ps = params()
    opt = O().AdamW(ps, state_bits=bits, capturable=True, **HYPER)
    for step in range(4):
        grads(ps, step)
        if step < 3:
            ps[1].grad = None
        opt.step()
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    again = O().AdamW(qs, state_bits=bits, capturable=True, lr=1.0)
    again.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert [int(again.state[q]['step']) for q in qs] == [4, 1, 4, 4] and again.param_groups[0]['step_count'].item() == 4
    grads(ps, 9), grads(qs, 9)
    opt.step(), again.step()
    assert all(torch.equal(p, q) for p, q in zip(ps, qs))
    old = copy.deepcopy(opt.state_dict())
    for s in old['state'].values():
        del s['step']
    again.load_state_dict(old)
    assert [int(again.state[q]['step']) for q in qs] == [5] * 4
    for group in opt.param_groups:
        group['capturable'] = False
    grads(ps, 10)
    opt.step()
    assert [opt.state[p]['step'] for p in ps] == [6, 3, 6, 6]
    for group in opt.param_groups:
        group['capturable'] = True
    opt.step()
    assert [int(opt.state[p]['step']) for p in ps] == [7, 4, 7, 7]


@pytest.mark.parametrize('bits', [8, 32])
def test_a_captured_step_goes_on_after_loading(bits):
    """Saved (to the host), loaded again and loaded with a state from before any step, a captured step with its learning rate on the
    device is replayed: bit for bit the eager run that loads the same."""
    import copy
    import io
    runs = []
    for captured in (True, False):
        ps = params()
        held = [torch.zeros_like(p) for p in ps]
        for p, h in zip(ps, held):
            p.grad = h
        opt = O().AdamW(ps, lr=torch.tensor(0.01, device=DEV), weight_decay=0.1, state_bits=bits, capturable=True)
        fresh = copy.deepcopy(opt.state_dict())
        opt.init_state()
        step = opt.step
        if captured:
            torch.cuda.synchronize()
            graph = torch.cuda.CUDAGraph()
            with torch.cuda.graph(graph):
                opt.step()
            step = graph.replay
        seen = []

        def go(n):
            for _ in range(n):
                g = torch.Generator().manual_seed(len(seen))
                for h in held:
                    h.copy_(torch.randn(h.shape, generator=g))
                step()
                torch.cuda.synchronize()
                seen.append([p.detach().clone() for p in ps])
                torch.randn(1 << 16, device=DEV)                           # takes what was given back to the allocator
        go(3)
        buf = io.BytesIO()
        torch.save(opt.state_dict(), buf)
        opt.param_groups[0]['lr'].fill_(0.5)
        go(2)
        buf.seek(0)
        opt.load_state_dict(torch.load(buf, weights_only=True, map_location='cpu'))
        go(3)
        assert opt.param_groups[0]['step_count'].item() == 6 and opt.param_groups[0]['lr'].item() == pytest.approx(0.01)
        opt.param_groups[0]['lr'].fill_(0.02)
        opt.load_state_dict(fresh)
        go(2)
        assert opt.param_groups[0]['step_count'].item() == 2 and [int(opt.state[p]['step']) for p in ps] == [2] * 4
        runs.append(seen)
    for a, b in zip(*runs):
        assert all(torch.equal(x, y) for x, y in zip(a, b))


@pytest.mark.parametrize('bits', [8, 32])
@pytest.mark.parametrize('uniform', [True, False])
def test_moments_in_two_places_are_refused(bits, uniform):
    """Tensors that a step writes belong to one parameter each: shared moments would be updated by two workgroups at once."""
    z = lambda n, d=torch.float32: torch.zeros(n, dtype=d, device=DEV)     # noqa: E731
    ps = [z(100), z(100, torch.float32 if uniform else torch.bfloat16)]
    gs = [torch.ones_like(p) for p in ps]
    one = lambda kind: z(100) if bits == 32 else (z(128, kind), z(1))       # noqa: E731
    ms, vs = [one(torch.int8) for _ in ps], [one(torch.uint8) for _ in ps]
    step = lambda m, v: O().adamw_step(ps, gs, m, v, step=1, lr=0.1)       # noqa: E731
    bad = [([ms[0]] * 2, vs), (ms, [vs[0]] * 2)]
    if bits == 32:
        bad += [([vs[0], ms[1]], vs), ([ps[0], ms[1]], vs)]
    else:
        bad += [([ms[0], (ms[1][0], ms[0][1])], vs), (ms, [(vs[0][0], ms[0][1]), vs[1]])]
    for m, v in bad:
        with pytest.raises(ValueError, match='twice'):
            step(m, v)
    assert not any(p.any() for p in ps)
    step(ms, vs)
    assert all(p.ne(0).all() for p in ps)


@pytest.mark.parametrize('dtype', DTYPES)
def test_8_bits_a_lost_element_changes_no_other(dtype):
    """NaN and infinite gradients, in a block whose scales do not hang on those elements: every other parameter, code and scale is bit
    for bit that of the run in which those elements have no moments and no gradient."""
    n, lost = 384, [3, 40, 255, 300]
    p, g = (t[0] for t in make([n], dtype)[:2])
    state = quantized([p])[0]
    for k in lost:
        state[0][k] = state[2][k] = 0
    bad, good = g.clone(), g.clone()
    bad[3], bad[40], bad[255], bad[300] = float('nan'), float('inf'), float('-inf'), float('nan')
    good[lost] = 0.0
    runs = []
    for grad in (bad, good):
        P, S = p.to(DEV), [x.clone().to(DEV) for x in state]
        for step in (7, 8, 9):                                              # lost in the first step, and not found again
            O().adamw_step([P], [(grad if step == 7 else good).to(DEV)], [(S[0], S[1])], [(S[2], S[3])], step=step, **HYPER)
        runs.append([P.cpu()] + [s.cpu() for s in S])
    keep = torch.ones(n, dtype=torch.bool)
    keep[lost] = False
    for a, b, what in zip(runs[0], runs[1], ('param', 'exp_avg', 'exp_avg scale', 'exp_avg_sq', 'exp_avg_sq scale')):
        rest = slice(None) if 'scale' in what else keep
        assert torch.equal(a[rest], b[rest]) and torch.isfinite(a[rest].float()).all(), what
    assert runs[0][1][lost].eq(-128).all() and runs[0][0][lost].isnan().all() and torch.isfinite(runs[1][0].float()).all()
