"""Embedding lookup and its gradient (csrc/embedding.hip) on the GPU against the plain 64-bit form of tests/training_ops.py.

Bounds: a row times a scale is one rounding in fp32 and one in the output type; a pooled row or a gradient row is a sum of n
products in fp32, off by at most (n + 2) roundings of the sum of absolute values, and one rounding in the output type."""
import pytest
import torch

from tests import training_ops as T

pytestmark = pytest.mark.gpu
DEV = 'cuda'
DTYPES = [torch.float32, torch.bfloat16, torch.float16]


def E():
    from ranking_amd import embedding
    return embedding


def make_ids(shape, rows, seed, dtype=torch.int64, pad=0.1, common=0.0):
    g = torch.Generator().manual_seed(seed)
    ids = torch.randint(0, max(rows, 1), shape, generator=g)
    ids[torch.rand(shape, generator=g) < common] = rows // 2
    ids[torch.rand(shape, generator=g) < pad] = -1
    return ids.to(dtype)


def check_lookup(table, ids, scale, combiner, what=''):
    out = E().embedding_lookup(table, ids, scale, combiner)
    want, size = T.embedding(table, ids, scale, combiner)
    assert out.dtype == table.dtype and out.is_contiguous()
    n = 0 if combiner is None else ids.shape[-1]
    T.assert_within(out, want, T.half(table.dtype) * want.abs().nan_to_num() * 1.001 + (n + 3) * T.U * size.nan_to_num() + T.tiny(table.dtype), what)
    return out


def check_grad(up, ids, rows, scale, combiner, what=''):
    got = E().embedding_grad(up, ids, rows, scale, combiner)
    want, size, count = T.embedding_gradient(up, ids, rows, scale, combiner)
    assert got.dtype == up.dtype and tuple(got.shape) == (rows, up.shape[-1])
    bound = T.half(up.dtype) * want.abs() * 1.001 + (count.unsqueeze(1) + 3) * T.U * size + T.tiny(up.dtype)
    T.assert_within(got, want, bound, what)
    return got


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('rows,dim,n', [(1, 1, 1), (5, 3, 7), (100, 20, 33), (50, 64, 1), (37, 130, 1000), (1000, 257, 65), (300, 1024, 129), (9, 4104, 5)])
def test_lookup_and_gradient(dtype, rows, dim, n):
    g = torch.Generator().manual_seed(rows + dim)
    table = torch.randn(rows, dim, generator=g).to(dtype).to(DEV)
    for id_dtype in (torch.int32, torch.int64):
        ids = make_ids((n,), rows, n, id_dtype).to(DEV)
        check_lookup(table, ids, 2.5, None)
        up = torch.randn(n, dim, generator=g).to(dtype).to(DEV)
        check_grad(up, ids, rows, 2.5, None)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('combiner', ['sum', 'mean'])
@pytest.mark.parametrize('rows,dim,bags,tokens', [(30, 20, 50, 8), (11, 7, 3, 1), (200, 64, 2, 333), (64, 33, 129, 5), (100, 512, 1, 1000), (8, 16, 5, 0)])
def test_pooled_lookup_and_gradient(dtype, combiner, rows, dim, bags, tokens):
    g = torch.Generator().manual_seed(dim + tokens)
    table = torch.randn(rows, dim, generator=g).to(dtype).to(DEV)
    ids = make_ids((bags, tokens), rows, tokens, torch.int32)
    ids[bags // 2] = -1                                                     # a bag that holds nothing
    ids = ids.to(DEV)
    out = check_lookup(table, ids, 0.5, combiner)
    assert not out[bags // 2].any()
    up = torch.randn(bags, dim, generator=g).to(dtype).to(DEV)
    check_grad(up, ids, rows, 0.5, combiner)


@pytest.mark.parametrize('n', [4096, 4097, 8192, 8193, 30001])
@pytest.mark.parametrize('rows', [3, 200, 257, 5000, 300007])
def test_gradient_sort_sizes(n, rows):
    """Both sorts, one, two and three digits, a token that is common."""
    ids = make_ids((n,), rows, n + rows, torch.int64, common=0.2).to(DEV)
    up = torch.randn(n, 8, generator=torch.Generator().manual_seed(n)).to(DEV)
    first = check_grad(up, ids, rows, 1.0, None)
    assert torch.equal(first, E().embedding_grad(up, ids, rows))            # the same bits again


@pytest.mark.parametrize('n,rows', [(32768, 700), (32769, 700), (40001, 70001), (1300001, 5003)])
def test_gradient_of_many_tiles(n, rows):
    """As many tiles as add each other's counts up, one more, and tiles of several parts; bags of three."""
    ids = make_ids((n,), rows, n, torch.int32, common=0.05).to(DEV)
    up = torch.randn(n, 4, generator=torch.Generator().manual_seed(n)).to(DEV)
    check_grad(up, ids, rows, 1.0, None)
    check_grad(up[:n // 3], ids[:n // 3 * 3].view(-1, 3), rows, 0.5, 'mean')


def test_gradient_table_with_three_digit_ids():
    rows, n = (1 << 20) + 5, 20000
    ids = make_ids((n,), rows, 3, common=0.1).to(DEV)
    ids[:2] = torch.tensor([rows - 1, 0], device=DEV)
    up = torch.randn(n, 4, generator=torch.Generator().manual_seed(3)).to(DEV)
    check_grad(up, ids, rows, 1.0, None)


@pytest.mark.parametrize('runs', [(63,), (64,), (65,), (127, 1), (128,), (129, 127), (255, 1, 256), (1000, 24, 3000), (20000, 1, 5)])
@pytest.mark.parametrize('dim', [8, 200])
def test_gradient_runs_across_chunks(runs, dim):
    """Runs of one token that end inside, on and behind a chunk."""
    ids = torch.cat([torch.full((c,), 2 * k + 1) for k, c in enumerate(runs)])
    ids = ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(5))].to(DEV)
    up = torch.randn(len(ids), dim, generator=torch.Generator().manual_seed(6)).to(DEV)
    check_grad(up, ids, 2 * len(runs) + 2, 1.0, None)


@pytest.mark.parametrize('combiner', [None, 'sum', 'mean'])
def test_padding_and_ids_beyond_the_table(combiner):
    table = torch.randn(6, 12, generator=torch.Generator().manual_seed(7)).to(DEV)
    ids = torch.tensor([[0, 5, -1], [6, 1, 2], [-7, -1, -9223372036854775808], [2, 9223372036854775807, 3]], device=DEV)
    out = check_lookup(table, ids, 1.0, combiner)
    assert out[2].eq(0).all() and out[1].isnan().any() and out[3].isnan().any() and not out[0].isnan().any()
    up = torch.randn((4, 3, 12) if combiner is None else (4, 12), generator=torch.Generator().manual_seed(8)).to(DEV)
    check_grad(up, ids, 6, 1.0, combiner)
    check_grad(up, torch.full_like(ids, -1), 6, 1.0, combiner)


def test_infinite_gradients_stay_in_their_row():
    ids = torch.tensor([1, 2, 1, -1, 5], device=DEV)
    up = torch.ones(5, 4, device=DEV)
    up[2, 1], up[3], up[4, 0] = float('inf'), float('nan'), float('nan')
    got = E().embedding_grad(up, ids, 5)
    assert got[1].tolist() == [2.0, float('inf'), 2.0, 2.0] and got[2].tolist() == [1.0] * 4
    assert not got[0].any() and not got[3].any() and not got[4].any()


@pytest.mark.parametrize('dtype', DTYPES)
def test_strides_and_alignments(dtype):
    """Tables that are a slice of a wider or a shifted buffer, ids and gradients of other strides."""
    g = torch.Generator().manual_seed(9)
    wide = torch.randn(20, 100, generator=g).to(dtype).to(DEV)
    ids = make_ids((6, 4), 20, 9).to(DEV)
    for table in (wide[:, 3:60], wide[:, 8:72], wide[::2, 1:33], wide.t()[:20, :15], wide.flatten()[1:20 * 30 + 1].view(20, 30)):
        i = ids.clamp(max=table.shape[0] - 1)
        check_lookup(table, i, 1.5, None)
        check_lookup(table, i, 1.5, 'mean')
        check_lookup(table, i.t(), 1.5, 'sum')
    up = torch.randn(6, 4, 200, generator=g).to(dtype).to(DEV)
    check_grad(up[:, :, 5:78], ids, 20, 1.0, None)
    check_grad(up[:, :1, 7:71].expand(6, 4, 64), ids, 20, 1.0, None)


def test_empty_calls():
    table = torch.randn(4, 8, device=DEV)
    none = torch.zeros(0, dtype=torch.int64, device=DEV)
    assert E().embedding_lookup(table, none).shape == (0, 8)
    assert E().embedding_lookup(table, none.view(3, 0), combiner='mean').eq(0).all()
    assert E().embedding_grad(torch.zeros(0, 8, device=DEV), none, 4).eq(0).all()
    assert E().embedding_grad(torch.zeros(0, 8, device=DEV), none, 0).shape == (0, 8)
    assert E().embedding_grad(torch.zeros(3, 8, device=DEV), none.view(3, 0), 4, combiner='sum').eq(0).all()
    assert E().embedding_lookup(torch.zeros(0, 8, device=DEV), torch.tensor([-1, 0], device=DEV))[1].isnan().all()
    assert E().embedding_lookup(table, torch.tensor(2, device=DEV)).shape == (8,)


def test_offsets_beyond_32_bits():
    """A table of 2^31 + elements: the last rows are read, and written by the gradient."""
    rows, dim = 2100000, 1040
    table = torch.empty(rows, dim, dtype=torch.bfloat16, device=DEV)
    ids = torch.tensor([rows - 1, 0, rows - 2], device=DEV)
    table[ids] = torch.arange(3 * dim, device=DEV).view(3, dim).to(torch.bfloat16)
    assert torch.equal(E().embedding_lookup(table, ids), table[ids])
    assert torch.equal(E().embedding_lookup(table, ids.view(1, 3)[:, :1], combiner='sum'), table[-1:])
    del table
    up = torch.ones(3, dim, dtype=torch.bfloat16, device=DEV)
    got = E().embedding_grad(up, ids, rows)
    assert got[ids].eq(1).all() and got.sum(dtype=torch.float64).item() == 3 * dim


@pytest.mark.parametrize('combiner', [None, 'mean'])
def test_autograd(combiner):
    g = torch.Generator().manual_seed(11)
    table = torch.randn(10, 6, generator=g).to(DEV).requires_grad_()
    ids = make_ids((5, 4), 10, 11).to(DEV)
    out = E().embedding_lookup(table, ids, 3.0, combiner)
    up = torch.randn(out.shape, generator=g).to(DEV)
    (out * up).sum().backward()
    assert torch.equal(table.grad, E().embedding_grad(up, ids, 10, 3.0, combiner))
    out = E().embedding_lookup(table, ids, 3.0, combiner)
    out.sum().backward()                                                    # an expanded upstream, added to what is there
    assert torch.allclose(table.grad, E().embedding_grad(up, ids, 10, 3.0, combiner) + E().embedding_grad(torch.ones_like(up), ids, 10, 3.0, combiner))
    with torch.no_grad():
        assert not E().embedding_lookup(table, ids).requires_grad


def test_other_stream():
    table = torch.randn(1000, 64, device=DEV)
    ids = make_ids((5000,), 1000, 12).to(DEV)
    up = torch.randn(5000, 64, device=DEV)
    want = E().embedding_lookup(table, ids), E().embedding_grad(up, ids, 1000)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        got = E().embedding_lookup(table, ids), E().embedding_grad(up, ids, 1000)
    torch.cuda.current_stream().wait_stream(s)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


@pytest.mark.parametrize('n', [100, 9000])
def test_captured_and_replayed(n):
    """Two graphs over the same inputs, replayed with new values in them and eager calls between."""
    table, up = torch.randn(500, 32, device=DEV), torch.randn(n, 32, device=DEV)
    ids = make_ids((n,), 500, 13, common=0.3).to(DEV)

    def step():
        return E().embedding_lookup(table, ids, 2.0), E().embedding_grad(up, ids, 500, 2.0)
    step()
    graphs = []
    for _ in range(2):
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out = step()
        graphs.append((g, out))
    for k in range(3):
        ids.copy_(make_ids((n,), 500, 20 + k, common=0.3))
        up.normal_()
        for g, _ in graphs:
            g.replay()
        want = step()
        torch.cuda.synchronize()
        for _, out in graphs:
            assert torch.equal(out[0], want[0]) and torch.equal(out[1], want[1])


def test_refusals():
    table, ids = torch.zeros(4, 8, device=DEV), torch.zeros(2, 3, dtype=torch.int64, device=DEV)
    for bad in (lambda: E().embedding_lookup(table.double(), ids), lambda: E().embedding_lookup(table, ids.float()),
                lambda: E().embedding_lookup(table, ids, combiner='max'), lambda: E().embedding_lookup(table[0], ids),
                lambda: E().embedding_lookup(table, ids[0, 0], combiner='sum'), lambda: E().embedding_grad(torch.zeros(2, 8, device=DEV), ids, 4),
                lambda: E().embedding_grad(torch.zeros(2, 3, 8, device=DEV), ids, -1),
                lambda: E().embedding_grad(torch.zeros(2, 3, 8, device=DEV), ids, 1 << 26),
                lambda: E().embedding_lookup(table, ids.new_zeros(1).expand(1 << 26))):
        with pytest.raises(ValueError):
            bad()


def test_layer_in_the_scorer():
    """DNNScorer with embedded context and example features = the same scorer fed with the embedded columns."""
    import ranking_amd as ra
    torch.manual_seed(0)
    L, M = ra.keras.layers, ra.keras.model
    emb = {'q': L.Embedding(50, 4, 'mean'), 'd': L.Embedding(30, 6, 'sum', 0.5), 'k': L.Embedding(9, 2, None)}
    scorer = M.DNNScorer(input_dim=4 + 6 + 2 * 3 + 5, embeddings=emb, hidden_layer_dims=[16], dropout=0.0, use_batch_norm=False).to(DEV)
    ctx = {'q': make_ids((3, 7), 50, 1).float().to(DEV)}
    ex = {'d': make_ids((3, 8, 5), 30, 2).to(DEV), 'k': make_ids((3, 8, 3), 9, 3, torch.int32).to(DEV), 'x': torch.randn(3, 8, 5, device=DEV)}
    mask = torch.ones(3, 8, dtype=torch.bool, device=DEV)
    mask[1, 5:] = False
    got = scorer(ctx, ex, mask)
    plain = M.DNNScorer(input_dim=21, hidden_layer_dims=[16], dropout=0.0, use_batch_norm=False).to(DEV)
    plain._tower.load_state_dict(scorer._tower.state_dict())
    dense_ctx = {'q': emb['q'](ctx['q'])}
    dense = {'d': emb['d'](ex['d']), 'k': emb['k'](ex['k']).flatten(2), 'x': ex['x']}
    assert torch.equal(got, plain(dense_ctx, dense, mask))
    got[mask].sum().backward()
    assert all(e.weight.grad is not None and e.weight.grad.abs().sum() > 0 for e in emb.values())


def test_the_most_lookups_of_a_call():
    """2^25 lookups of rows that take two column steps of a wavefront: 2^24 workgroups and more in all, in launches that hold them."""
    n, dim, rows = 1 << 25, 65, 1000
    table = torch.randn(rows, dim, generator=torch.Generator().manual_seed(1)).to(torch.bfloat16).to(DEV)
    ids = torch.randint(0, rows, (n,), generator=torch.Generator(device=DEV).manual_seed(2), device=DEV, dtype=torch.int32)
    ids[-1], ids[0] = 7, -1
    out = E().embedding_lookup(table, ids)
    assert not out[0].any()
    for a in range(0, n, 1 << 22):
        at = ids[a:a + (1 << 22)].long()
        assert torch.equal(out[a:a + (1 << 22)][at >= 0], table[at[at >= 0]])


def test_gradient_of_wide_bags():
    """Rows of 2^20 - 1 numbers, 65 535 occurrences in 255 bags: 2^24 workgroups for the runs.  In float64 by column parts."""
    bags, tokens, dim, rows = 255, 257, (1 << 20) - 1, 512
    ids = make_ids((bags, tokens), rows, 5, torch.int32, pad=0.05).to(DEV)
    up = torch.randn(bags, dim, generator=torch.Generator(device=DEV).manual_seed(6), device=DEV).to(torch.bfloat16)
    got = E().embedding_grad(up, ids, rows, 0.5, 'sum')
    count = torch.zeros(rows + 1, bags, dtype=torch.float64, device=DEV)
    at = torch.where(ids >= 0, ids.long(), rows)
    count.index_put_((at, torch.arange(bags, device=DEV).unsqueeze(1).expand_as(at)), torch.ones((), dtype=torch.float64, device=DEV), accumulate=True)
    count = count[:-1]
    most = count.sum(1, keepdim=True)
    for a in range(0, dim, 1 << 17):
        u = up[:, a:a + (1 << 17)].double()
        want, size = 0.5 * (count @ u), 0.5 * (count @ u.abs())
        off = (got[:, a:a + (1 << 17)].double() - want).abs() - (2.0 ** -8 * 1.001 * want.abs() + (most + 3) * T.U * size)
        assert off.max() <= 0


# ---------------------------------------------------------------- sizes that take other paths
def runs_of(lengths, seed, pad=0):
    """Ids in a random order: token 2 k + 1 occurs lengths[k] times, `pad` more are padding."""
    ids = torch.cat([torch.full((c,), 2 * k + 1, dtype=torch.int32) for k, c in enumerate(lengths)] + [torch.full((pad,), -1, dtype=torch.int32)])
    return ids[torch.randperm(len(ids), generator=torch.Generator().manual_seed(seed))].to(DEV)


def borders(chunk, n):
    """Run lengths of n occurrences in all: runs that begin and end on, before and behind borders of chunks of `chunk`, one of 16 chunks
    and more, many of one and two."""
    runs = [chunk, chunk - 1, chunk + 1, 1, chunk - 1, 2 * chunk, 2 * chunk + 1, chunk - 2, 1, 16 * chunk, 15 * chunk, 17 * chunk + 3, 40 * chunk - 3]
    left = n - sum(runs)
    assert left > 0
    runs += [left // 4] + [2, 1] * (left // 8) + [5] * (left // 32)
    return runs + [n - sum(runs)]


@pytest.mark.parametrize('dim,dtype', [(300, torch.float32), (300, torch.bfloat16), (1001, torch.float32), (1001, torch.bfloat16), (1024, torch.float16)])
def test_gradient_of_long_runs_in_wide_rows(dim, dtype):
    """Runs of 16 chunks and more, joined by a whole workgroup, in rows of several column steps; the same bits on repeat."""
    lengths = [16 * 16 + 1, 15 * 16, 3, 17 * 16 - 1, 700, 1, 5]
    ids = runs_of(lengths, 1, pad=9)
    up = torch.randn(len(ids), dim, generator=torch.Generator().manual_seed(dim)).to(dtype).to(DEV)
    rows = 2 * len(lengths) + 1
    first = check_grad(up, ids, rows, 1.5, None)
    assert torch.equal(first, E().embedding_grad(up, ids, rows, 1.5))
    bags = len(ids) // 4
    check_grad(up[:bags], ids[:4 * bags].view(bags, 4), rows, 1.5, 'mean')


# a chunk doubles while the next length times 131 072 is within n times the lanes of a row: 32 from 65 536 occurrences of 64 lanes on,
# 64 from 131 072, 128 beyond 2^20 occurrences
@pytest.mark.parametrize('chunk,n,dim', [(16, 65535, 256), (32, 65537, 256), (64, 131073, 256), (64, 140001, 260), (128, 1100003, 64), (128, 1100003, 100)])
def test_gradient_of_long_chunks(chunk, n, dim):
    """Every length of a chunk: small integers, whose sums fp32 holds exactly, against the same sums in float64."""
    lengths = borders(chunk, n - 777)
    ids, rows = runs_of(lengths, chunk, pad=777), 2 * len(lengths) + 1
    up = torch.randint(-8, 9, (n, dim), generator=torch.Generator(device=DEV).manual_seed(n), device=DEV).float()
    got = E().embedding_grad(up, ids, rows)
    at = torch.where(ids >= 0, ids.long(), rows)
    want = torch.zeros(rows + 1, dim, dtype=torch.float64, device=DEV).index_add_(0, at, up.double())[:-1]
    assert torch.equal(got.double(), want)
    if dim == 256:                                                          # bf16: sums in fp32, one rounding
        assert torch.equal(E().embedding_grad(up.to(torch.bfloat16), ids, rows), want.to(torch.bfloat16))
    bags = n // 11
    pooled = E().embedding_grad(up[:bags], ids[:bags * 11].view(bags, 11), rows, combiner='sum')
    want = torch.zeros(rows + 1, dim, dtype=torch.float64, device=DEV).index_add_(0, at[:bags * 11], up[:bags].double().repeat_interleave(11, 0))[:-1]
    assert torch.equal(pooled.double(), want)


@pytest.mark.parametrize('dtype', DTYPES)
@pytest.mark.parametrize('dim', [512, 514, 513])
def test_lookup_beyond_the_caches(dtype, dim):
    """Results of more than 32 MB go past the caches: 16-byte, 4-byte and single elements a lane; the same bits as row by row."""
    n, rows = 70001, 3001
    table = torch.randn(rows, dim, generator=torch.Generator(device=DEV).manual_seed(dim), device=DEV).to(dtype)
    ids = make_ids((n,), rows, dim).to(DEV)
    ids[5] = rows
    assert n * dim * table.element_size() > 32 << 20
    out = E().embedding_lookup(table, ids, 0.5)
    want = (table.float()[ids.clamp(0, rows - 1)] * 0.5).to(dtype)
    want[ids < 0] = 0
    assert out[5].isnan().all()
    keep = torch.arange(n, device=DEV) != 5
    assert torch.equal(out[keep], want[keep])
    assert torch.equal(out[:1000][keep[:1000]], E().embedding_lookup(table, ids[:1000], 0.5)[keep[:1000]])


@pytest.mark.parametrize('dim,dtype', [(1024, torch.bfloat16), (1022, torch.bfloat16), (1023, torch.bfloat16), (640, torch.float32)])
def test_gradient_table_beyond_the_caches(dim, dtype):
    """A table of more than 256 MB, written past the caches, of many lookups; small integers as above."""
    rows, n = 140001, 90001
    ids = make_ids((n,), rows, dim, torch.int32, common=0.1).to(DEV)
    up = torch.randint(-8, 9, (n, dim), generator=torch.Generator(device=DEV).manual_seed(dim), device=DEV).to(dtype)
    assert rows * dim * up.element_size() > 256 << 20
    got = E().embedding_grad(up, ids, rows)
    at = torch.where(ids >= 0, ids.long(), rows)
    want = torch.zeros(rows + 1, dim, device=DEV).index_add_(0, at, up.float())[:-1]      # exact: integers below 2^24 in any order
    assert torch.equal(got, want.to(dtype))


@pytest.mark.parametrize('padded', [False, True])
@pytest.mark.parametrize('dtype', [torch.float32, torch.bfloat16])
def test_layer_in_front_of_the_fused_tower(dtype, padded):
    """DNNScorer's bf16 tower behind embedded example features: logits and table gradients are those of the same tower fed with the
    embedded columns, the columns' gradient brought to the table by embedding_grad."""
    import ranking_amd as ra
    from ranking_amd.tower import FusedTower
    torch.manual_seed(0)
    L, M = ra.keras.layers, ra.keras.model
    emb = {'d': L.Embedding(60, 24, 'mean', dtype=dtype), 'k': L.Embedding(9, 8, None, dtype=dtype)}
    kw = dict(input_dim=24 + 8 * 3, hidden_layer_dims=[64, 32], dropout=0.0, compute_dtype=torch.bfloat16)
    scorer, plain = M.DNNScorer(embeddings=emb, **kw).to(DEV), M.DNNScorer(**kw).to(DEV)
    assert isinstance(scorer._tower, FusedTower)
    plain._tower.load_state_dict(scorer._tower.state_dict())
    ids = {'d': make_ids((16, 20, 5), 60, 2).to(DEV), 'k': make_ids((16, 20, 3), 9, 3, torch.int32).to(DEV)}
    mask = torch.ones(16, 20, dtype=torch.bool, device=DEV)
    if padded:
        mask[:, 13:] = False
        mask[3, 2:] = False
    up = torch.randn(16, 20, generator=torch.Generator().manual_seed(4)).to(DEV) * mask
    got = scorer({}, ids, mask)
    got.backward(up)
    dense = {k: emb[k](v).detach().flatten(2).requires_grad_() for k, v in ids.items()}
    want = plain({}, dense, mask)
    want.backward(up)
    assert torch.equal(got, want) and got[mask].abs().sum() > 0
    for k, combiner in (('d', 'mean'), ('k', None)):
        g = dense[k].grad if combiner else dense[k].grad.view(16, 20, 3, 8)
        wide, size, count = T.embedding_gradient(g, ids[k], emb[k].num_embeddings, 1.0, combiner)
        assert wide.abs().sum() > 0
        # padded lists: rows that are scored several times are added by atomics, in any order: 20 roundings of fp32, or of a bf16 step
        again = (20 * T.U if dtype == torch.float32 else 2 * T.half(dtype)) * size if padded else 0.0
        T.assert_within(emb[k].weight.grad, wide, T.half(dtype) * wide.abs() * 1.001 + (count.unsqueeze(1) + 3) * T.U * size + again + T.tiny(dtype), k)
