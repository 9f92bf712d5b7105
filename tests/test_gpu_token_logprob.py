"""Token log probabilities and their gradient (csrc/token_logprob.hip) on the GPU against the plain 64-bit form; the bounds are
derived in tests/training_ops.py (log_probs_bounds)."""
import pytest
import torch

from tests import training_ops as T

pytestmark = pytest.mark.gpu
DEV = 'cuda'
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def P():
    from ranking_amd import preference
    return preference


def check(logits, targets, temperature=1.0, upstream=None):
    logp, stats = P().token_log_probs_with_stats(logits, targets, temperature)
    assert logp.dtype == torch.float32 and logp.shape == targets.shape
    assert torch.equal(logp.nan_to_num(nan=7.0), P().token_log_probs(logits, targets, temperature).nan_to_num(nan=7.0))
    want = T.log_probs(logits, targets, temperature)
    bound, rel = T.log_probs_bounds(logits, targets, temperature)
    T.assert_within(logp, want, bound, 'log probabilities')
    if upstream is None:
        upstream = torch.randn(targets.shape, generator=torch.Generator().manual_seed(1)).to(DEV)
    got = P().token_log_probs_grad(upstream, logits, targets, stats, temperature)
    assert got.dtype == logits.dtype and got.shape == logits.shape and got.is_contiguous()
    want, p = T.log_probs_gradient(upstream, logits, targets, temperature)
    up = upstream.double().cpu().abs().unsqueeze(-1) / temperature
    d = (logits.double().cpu().clamp(min=-1e30) - logits.double().cpu().amax(-1, keepdim=True).clamp(-1e30)).abs() / temperature
    # the probability: the sum's error, its own argument's (3 U d) and 4 roundings more; the target's difference and the type's one
    bound = up * p.nan_to_num() * (rel.unsqueeze(-1) + (3 * d.clamp(max=110) + 6) * T.U) + 3 * T.U * up
    bound = bound.nan_to_num() + T.half(logits.dtype) * want.abs().nan_to_num() * 1.001 + T.tiny(logits.dtype)
    T.assert_within(got, want, bound, 'gradient')
    return logp, got


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('n,vocab', [(1, 1), (3, 2), (5, 7), (4, 64), (9, 200), (2, 2048), (3, 2049), (2, 5003), (1, 40000), (2, 100003), (700, 2100), (1000, 6), (333, 70), (77, 300)])
def test_sizes(dtype, n, vocab):
    g = torch.Generator().manual_seed(vocab)
    logits = (torch.randn(n, vocab, generator=g) * 4).to(dtype).to(DEV)
    targets = torch.randint(0, vocab, (n,), generator=g)
    if n > 2:
        targets[1] = -1
    for temperature in (1.0, 0.5):
        check(logits, targets.to(DEV), temperature)


def test_no_target_and_targets_beyond():
    logits = torch.randn(5, 30, generator=torch.Generator().manual_seed(2)).to(DEV)
    logits[0] = float('nan')                                               # a row that is no target is not read
    targets = torch.tensor([-1, 30, 29, -5, 9223372036854775807], device=DEV)
    logp, grad = check(logits, targets)
    assert logp[0] == 0 and logp[1].isnan() and logp[4].isnan() and grad[0].eq(0).all() and grad[1].isnan().all()
    big = torch.randn(3, 9000, device=DEV)
    big[1] = float('nan')
    logp, grad = check(big, torch.tensor([4, -1, 9000], device=DEV))
    assert logp[1] == 0 and grad[1].eq(0).all() and grad[2].isnan().all()


@pytest.mark.parametrize('vocab', [50, 5000, 70000])
@pytest.mark.parametrize('dtype', DTYPES)
def test_masked_logits(vocab, dtype):
    """-inf and the type's lowest value in masked places, all but one, and a row of -inf (NaN, as its softmax is)."""
    g = torch.Generator().manual_seed(vocab)
    logits = torch.randn(5, vocab, generator=g).to(dtype)
    low = torch.finfo(dtype).min
    logits[0, vocab // 2:] = -float('inf')
    logits[1, : vocab // 2] = low
    logits[2, :], logits[2, 3] = -float('inf'), 1.5
    logits[3, :], logits[3, 3] = low, 1.5
    targets = torch.tensor([vocab // 2, vocab - 1, 3, 3, 0])               # one masked target: -inf
    logp, grad = check(logits.to(DEV), targets.to(DEV))
    assert logp[0] == -float('inf') and logp[2] == 0 and logp[3] == 0
    logits[4] = low                                                        # all at the lowest value: uniform
    check(logits.to(DEV), targets.to(DEV))
    logits[4] = -float('inf')
    logp, stats = P().token_log_probs_with_stats(logits.to(DEV), targets.to(DEV))
    assert logp[4].isnan() and not logp[1:4].isnan().any()


def test_infinite_and_nan_logits():
    logits = torch.zeros(3, 100, device=DEV)
    logits[0, 5], logits[1, 7] = float('inf'), float('nan')
    assert P().token_log_probs(logits, torch.tensor([5, 7, 2], device=DEV)).isnan().tolist() == [True, True, False]


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('vocab', [101, 4099])
def test_strides(dtype, vocab):
    """The shifted slice of [batch, time, vocab], slices of wider rows, transposes and one row for all."""
    g = torch.Generator().manual_seed(5)
    x = torch.randn(3, 6, vocab + 9, generator=g).to(dtype).to(DEV)
    t = torch.randint(0, vocab - 5, (3, 6), generator=g).to(DEV)
    check(x[:, :-1, :], t[:, 1:])
    check(x[:, 1:, 3:vocab], t[:, 1:])
    check(x.transpose(0, 1)[:, :, :vocab], t.t())
    check(x[:, ::2, :vocab], t[:, ::2])
    check(x[:1, :1].expand(3, 6, vocab + 9), t)
    check(x[0, 0], t[0, 0])
    check(x.permute(2, 0, 1)[: vocab - 5, :, :4], torch.zeros(vocab - 5, 3, dtype=torch.int64, device=DEV))
    check(x.view(3, 2, 3, -1), t.view(3, 2, 3).to(torch.int32))
    check(x.flatten()[1:1 + 4 * vocab].view(4, vocab), t.flatten()[:4])


def test_zero_upstream_and_empty():
    x, t = torch.randn(4, 50, device=DEV), torch.tensor([1, 2, 3, 4], device=DEV)
    _, grad = check(x, t, upstream=torch.tensor([0.0, 1.0, -2.0, 0.0], device=DEV))
    assert not grad[0].any() and not grad[3].any()
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    assert P().token_log_probs(torch.zeros(0, 9, device=DEV), none).shape == (0,)
    logp, stats = P().token_log_probs_with_stats(torch.zeros(2, 0, 9, device=DEV), none.view(2, 0))
    assert P().token_log_probs_grad(logp, torch.zeros(2, 0, 9, device=DEV), none.view(2, 0), stats).shape == (2, 0, 9)


def test_autograd_against_differences():
    g = torch.Generator().manual_seed(6)
    x = torch.randn(2, 3, 12, generator=g).to(DEV).requires_grad_()
    t = torch.randint(0, 12, (2, 3), generator=g).to(DEV)
    up = torch.randn(2, 3, generator=g).to(DEV)
    (P().token_log_probs(x, t, 0.8) * up).sum().backward()
    h = 2.0 ** -7
    with torch.no_grad():
        for at in [(0, 0, 0), (1, 2, 11), (0, 1, int(t[0, 1]))]:
            hi, lo = x.detach().clone(), x.detach().clone()
            hi[at] += h
            lo[at] -= h
            diff = ((P().token_log_probs(hi, t, 0.8).double() - P().token_log_probs(lo, t, 0.8).double()) * up).sum() / (2 * h)
            # curvature: h^2 / 6 |f'''| <= h^2 / 6 |up| / T^3 / 4 < 1e-4; rounding: 2^-22 values / 2^-6 < 1e-4
            assert abs(diff - x.grad[at]) < 2e-4 + 2e-4


def test_offsets_beyond_32_bits():
    n, vocab = 70000, 66000                                                # 4.6e9 elements
    x = torch.zeros(n, vocab, dtype=torch.bfloat16, device=DEV)
    x[n - 1, vocab - 1] = 3.0
    t = torch.full((n,), -1, device=DEV)
    t[n - 1] = vocab - 1
    logp, stats = P().token_log_probs_with_stats(x, t)
    want = 3.0 - torch.log(torch.tensor(vocab - 1 + 2.718281828459045 ** 3, dtype=torch.float64)).item()
    assert abs(logp[n - 1].item() - want) < 1e-5 and not logp[:-1].any()
    grad = P().token_log_probs_grad(torch.ones(n, device=DEV), x, t, stats)
    assert grad[n - 1, vocab - 1] > 0.99 and not grad[n - 2].any() and grad[n - 1, 0] < 0


def test_logits_beyond_the_caches():
    """300 MB of logits go past the caches: the same bits as the same rows alone."""
    x = torch.randn(1500, 100003, dtype=torch.bfloat16, device=DEV)
    t = torch.randint(-1, 100003, (1500,), generator=torch.Generator().manual_seed(8)).to(DEV)
    up = torch.randn(1500, device=DEV)
    logp, stats = P().token_log_probs_with_stats(x, t)
    grad = P().token_log_probs_grad(up, x, t, stats)
    for rows in (slice(0, 600), slice(900, 1500)):
        part, part_stats = P().token_log_probs_with_stats(x[rows], t[rows])
        assert torch.equal(part, logp[rows]) and torch.equal(part_stats, stats[rows])
        assert torch.equal(P().token_log_probs_grad(up[rows], x[rows], t[rows], part_stats), grad[rows])
    check(x[3:6, 1:], t[3:6].clamp(max=100001), upstream=up[3:6])


def test_other_stream_and_graphs():
    x, t = torch.randn(6, 50000, device=DEV), torch.tensor([1, -1, 3, 4, 5, 6], device=DEV)
    up = torch.randn(6, device=DEV)

    def step():
        logp, stats = P().token_log_probs_with_stats(x, t)
        return logp, P().token_log_probs_grad(up, x, t, stats)
    want = step()
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = step()
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for _ in range(3):
        x.normal_()
        graph.replay()
        want = step()
        torch.cuda.synchronize()
        assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals():
    x, t = torch.zeros(4, 8, device=DEV), torch.zeros(4, dtype=torch.int64, device=DEV)
    for bad in (lambda: P().token_log_probs(x.double(), t), lambda: P().token_log_probs(x, t.float()), lambda: P().token_log_probs(x, t[:3]),
                lambda: P().token_log_probs(x, t, temperature=0.0), lambda: P().token_log_probs(x, t, temperature=float('nan')),
                lambda: P().token_log_probs(x[:, :0], t),
                lambda: P().token_log_probs_grad(t[:3].float(), x, t, torch.zeros(4, 2, device=DEV)),
                lambda: P().token_log_probs_grad(t.float(), x, t, torch.zeros(4, 3, device=DEV)),
                lambda: P().token_log_probs(x.new_zeros(1, 1).expand(1 << 24, 1), t.new_zeros(1).expand(1 << 24))):
        with pytest.raises(ValueError):
            bad()
