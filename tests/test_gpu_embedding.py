"""efgs.embedding on the GPU against the 64-bit oracle (oracle/training_ref.py).

Bars, e = 2^-24: a looked-up value is one float32 product rounded once to its type, so it equals torch's (table.float() * scale)
cast to that type bit for bit. A row's gradient is a float32 sum of its k upstream rows in some order, at most (k + 1) e of the sum
of their magnitudes off (k - 1 additions, the product, a last rounding), and half a step of the type, e, 2^-8 or 2^-11 of
the value (float16: and half its least step, 2^-25).
"""
import numpy as np
import pytest
import torch

import training_ref as R

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = {'f32': (torch.float32, E, 0.0), 'bf16': (torch.bfloat16, 2.0 ** -8, 0.0), 'f16': (torch.float16, 2.0 ** -11, 2.0 ** -25)}
DEVICE = 'cuda:0'


def _inputs(n, rows, columns, dtype, seed=0, skew=2.0, invalid=0.05, index=torch.int64):
    rng = np.random.default_rng(seed)
    indices = np.minimum((rows * rng.random(n) ** skew).astype(np.int64), max(rows - 1, 0))
    wrong = np.array([-1, rows, rows + 5, -(1 << 31), (1 << 31) - 1])
    pick = rng.random(n) < invalid
    indices[pick] = wrong[rng.integers(0, 5, int(pick.sum()))]
    kind = TYPES[dtype][0]
    table = torch.tensor(rng.normal(size=(rows, columns)), device=DEVICE).to(kind).requires_grad_()
    grad = torch.tensor(rng.normal(size=(n, columns)), device=DEVICE).to(kind)
    return torch.tensor(indices, device=DEVICE).to(index), table, grad


def _plain(indices, table, scale):
    rows = table.shape[0]
    inside = (indices >= 0) & (indices < rows)
    out = table.detach().float()[indices.long().clamp(0, max(rows - 1, 0))] * scale
    return torch.where(inside[..., None], out, torch.zeros_like(out)).to(table.dtype)


def _check_gradient(got, indices, grad, rows, scale, dtype, padding=None):
    want, size, entries = R.embedding_gradient(indices.cpu().numpy(), grad.double().cpu().numpy(), rows, scale, padding)
    got = got.double().cpu().numpy()
    _, rounding, least = TYPES[dtype]
    bound = (entries[:, None] + 1) * E * size + rounding * np.abs(want) * (1 + 1e-6) + least
    off = np.abs(got - want)
    assert np.all(off <= bound), (np.max(off / np.maximum(bound, 1e-300)), np.unravel_index(np.argmax(off - bound), off.shape))
    assert np.all(got[entries == 0] == 0.0)


def _check(n, rows, columns, dtype, scale=1.7, padding=None, **how):
    import efgs
    print(f'case embedding n={n} rows={rows} columns={columns} {dtype} {how}', flush=True)
    indices, table, grad = _inputs(n, rows, columns, dtype, **how)
    out = efgs.embedding(indices, table, scale, padding)
    assert out.shape == (n, columns) and out.dtype == table.dtype
    assert torch.equal(out, _plain(indices, table, scale))
    out.backward(grad)
    assert table.grad.dtype == table.dtype
    _check_gradient(table.grad, indices, grad, rows, scale, dtype, padding)
    return indices, table, grad


@pytest.mark.parametrize('columns', [1, 2, 3, 4, 5, 7, 8, 9, 16, 17, 31, 45, 64, 100, 129, 255, 257, 513, 1000, 1025, 2051, 4100, 8200])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_widths(columns, dtype):
    _check(301, 67, columns, dtype, seed=columns)


@pytest.mark.parametrize('n', [1, 2, 63, 64, 65, 255, 1023, 1024, 1025, 4095, 4096, 4097, 12_345, 70_001])
@pytest.mark.parametrize('rows', [1, 2, 255, 256, 257, 5000])
def test_lengths_and_rows(n, rows):
    _check(n, rows, 5, 'f32', seed=n + rows, padding=min(1, rows - 1))


@pytest.mark.parametrize('rows', [65_535, 65_536, 70_000, 1_000_000])
@pytest.mark.parametrize('n', [1, 1000, 30_000])
def test_large_tables(rows, n):
    _check(n, rows, 8, 'bf16', seed=n, skew=1.0)


@pytest.mark.parametrize('index', [torch.int32, torch.int64])
def test_index_types(index):
    _check(5000, 300, 12, 'f32', index=index)


@pytest.mark.parametrize('n, rows, columns, dtype', [(100_000, 1, 8, 'f32'), (100_000, 3, 1, 'f32'), (60_000, 1, 300, 'bf16'), (20_000, 2, 1030, 'f16'),
                                                     (300_000, 1, 3, 'f32')])
def test_rows_met_by_nearly_every_index(n, rows, columns, dtype):
    """One row crosses every block, with the carries of hundreds of them."""
    _check(n, rows, columns, dtype, skew=1.0, invalid=0.001)


@pytest.mark.parametrize('n, rows, columns, dtype', [(262_144, 4096, 8, 'f32'), (262_145, 4096, 8, 'f32'), (300_001, 257, 45, 'f32'), (524_289, 511, 4, 'f32'),
                                                     (530_000, 512, 3, 'f32'), (1_048_577, 300, 8, 'bf16'), (1_100_000, 4096, 8, 'f32'), (4000, 4096, 8, 'f16'),
                                                     (4000, 4097, 8, 'f16'), (9000, 1024, 64, 'f32'), (9000, 1025, 64, 'f32'), (1500, 4095, 16, 'f32'),
                                                     (20_000, 1000, 128, 'bf16'), (70_000, 64, 7, 'bf16'), (5000, 40, 68, 'f32')])
def test_small_tables_and_their_limits(n, rows, columns, dtype):
    """Tables summed by tiles, and just past that: one, two and four keys a thread, several tiles to a block, one and two passes of the
    tile's sort, the largest number of rows, the largest table, the widest rows."""
    _check(n, rows, columns, dtype, seed=n % 1000, padding=3)


@pytest.mark.parametrize('n, rows, columns', [(150_000, 6000, 3), (300_000, 5000, 8), (1_200_000, 4200, 2), (1_060_000, 70_000, 1)])
def test_long_lists_into_larger_tables(n, rows, columns):
    """The list in order over the GPU: several tiles to a block of its passes, digits of 7 to 9 bits, hot rows among many."""
    _check(n, rows, columns, 'f32', skew=3.0)


@pytest.mark.parametrize('rows', [4500, 100_000])
def test_one_row_met_by_nearly_all_of_a_larger_table(rows):
    import efgs
    n = 120_000
    indices = torch.full((n,), rows // 2, device=DEVICE)
    indices[::500] = torch.randint(0, rows, (n // 500,), device=DEVICE)
    grad = torch.randn(n, 12, device=DEVICE)
    table = torch.zeros(rows, 12, device=DEVICE, requires_grad=True)
    got = torch.autograd.grad(efgs.embedding(indices, table, 0.5), table, grad)[0]
    _check_gradient(got, indices, grad, rows, 0.5, 'f32')


@pytest.mark.parametrize('n, rows, columns, dtype', [(131_002, 70, 130, 'f32'), (131_003, 70, 130, 'f32'), (131_066, 70, 513, 'bf16'), (150_000, 5000, 256, 'f32'), (300_001, 5000, 130, 'f32')])
@pytest.mark.parametrize('hot, share', [(0, 1.0), (69, 1.0), (17, 0.97), (17, 0.5), (5, 0.1)])
def test_rows_that_run_over_many_blocks(n, rows, columns, dtype, hot, share):
    """Small whole numbers, whose sums are exact in any order: a part of a row that is lost or counted twice shows. (The sums are of less
    than 2^24 in float32; bfloat16 rounds them once.) Lists of 131,072 entries and rows on begin the sum in chunks."""
    import efgs
    print(f'case embedding hot n={n} rows={rows} columns={columns} {dtype} hot={hot} share={share}', flush=True)
    generator = torch.Generator(device=DEVICE).manual_seed(n + hot)
    indices = torch.randint(-1, rows + 1, (n,), device=DEVICE, generator=generator)
    indices[torch.rand(n, device=DEVICE, generator=generator) < share] = hot
    grad = torch.randint(-4, 8, (n, columns), device=DEVICE, generator=generator)
    table = torch.zeros(rows, columns, dtype=TYPES[dtype][0], device=DEVICE, requires_grad=True)
    efgs.embedding(indices, table).backward(grad.to(table.dtype))
    others = (indices >= 0) & (indices < rows) & (indices != hot)
    want = torch.zeros(rows, columns, dtype=torch.float64, device=DEVICE).index_add_(0, indices[others], grad[others].double())
    want[hot] = grad[indices == hot].sum(0).double()
    assert torch.equal(table.grad, want.to(table.dtype))


def test_hot_row_between_empty_ones():
    import efgs
    n, rows = 50_000, 9000
    indices = torch.full((n,), 4500, device=DEVICE)
    indices[::1000] = torch.arange(50, device=DEVICE) * 180
    grad = torch.randn(n, 16, device=DEVICE)
    table = torch.randn(rows, 16, device=DEVICE, requires_grad=True)
    efgs.embedding(indices, table).backward(grad)
    _check_gradient(table.grad, indices, grad, rows, 1.0, 'f32')


@pytest.mark.parametrize('rows, columns, dtype', [(60_001, 513, 'f32'), (100_003, 1024, 'bf16'), (13_000_001, 5, 'f16')])
def test_gradient_of_a_table_that_no_cache_holds(rows, columns, dtype):
    """Gradients of over 100 MB (stored past the caches), most rows zero; against sums in 64 bits on the GPU."""
    import efgs
    print(f'case embedding large table {rows} x {columns} {dtype}', flush=True)
    kind, rounding, least = TYPES[dtype]
    table = torch.zeros((rows, columns), dtype=kind, device=DEVICE, requires_grad=True)
    indices = torch.randint(0, rows, (9001,), device=DEVICE)
    indices[::3] = rows - 1
    grad = torch.randn(9001, columns, device=DEVICE).to(kind)
    got = torch.autograd.grad(efgs.embedding(indices, table, 1.5), table, grad)[0]
    met, where, entries = torch.unique(indices, return_inverse=True, return_counts=True)
    want = torch.zeros((len(met), columns), dtype=torch.float64, device=DEVICE).index_add_(0, where, grad.double()) * 1.5
    size = torch.zeros((len(met), columns), dtype=torch.float64, device=DEVICE).index_add_(0, where, grad.double().abs()) * 1.5
    bound = (entries[:, None] + 1) * E * size + rounding * want.abs() * (1 + 1e-6) + least
    assert bool(((got[met].double() - want).abs() <= bound).all())
    got[met] = 0
    assert not bool(got.any())


def test_more_indices_than_a_pass_of_the_sort_takes_at_once():
    """Over a million indices: several tiles to a block of the sort."""
    _check(2_200_003, 3000, 1, 'f32')


def test_no_indices_no_valid_ones_no_rows():
    import efgs
    table = torch.randn(40, 6, device=DEVICE, requires_grad=True)
    out = efgs.embedding(torch.zeros(0, dtype=torch.int64, device=DEVICE), table)
    assert out.shape == (0, 6)
    assert torch.equal(torch.autograd.grad(out.sum(), table)[0], torch.zeros_like(table))
    out = efgs.embedding(torch.full((500,), -1, device=DEVICE), table)
    assert torch.equal(out, torch.zeros_like(out))
    assert torch.equal(torch.autograd.grad(out.sum(), table)[0], torch.zeros_like(table))
    empty = torch.zeros(0, 6, device=DEVICE, requires_grad=True)
    out = efgs.embedding(torch.zeros(3, dtype=torch.int64, device=DEVICE), empty)
    assert torch.equal(out, torch.zeros(3, 6, device=DEVICE))
    assert torch.autograd.grad(out.sum(), empty)[0].shape == (0, 6)
    assert efgs.embedding(torch.zeros(3, dtype=torch.int64, device=DEVICE), torch.zeros(4, 0, device=DEVICE)).shape == (3, 0)


def test_shapes_strides_and_alignment():
    """Indices of several dimensions and strides, tables of wide rows, turned tables, tables and upstream gradients that begin anywhere."""
    import efgs
    rng = torch.Generator(DEVICE).manual_seed(0)
    indices = torch.randint(0, 50, (6, 7, 8), generator=rng, device=DEVICE).permute(2, 0, 1)
    wide = torch.randn(50, 40, generator=rng, device=DEVICE)
    for name, table in (('slice', wide[:, 3:20]), ('turned', torch.randn(17, 50, generator=rng, device=DEVICE).T), ('every second', wide[:, ::2]),
                        ('one row for all', wide[:1].expand(50, 40)), ('offset', torch.randn(50 * 9 + 1, generator=rng, device=DEVICE).bfloat16()[1:].view(50, 9))):
        print('case embedding table', name, flush=True)
        leaf = table.detach().requires_grad_()
        out = efgs.embedding(indices, leaf, 0.5)
        assert out.shape == (8, 6, 7, table.shape[1]) and torch.equal(out, _plain(indices, table, 0.5))
        grad = torch.randn(out.numel() + 1, generator=rng, device=DEVICE).to(table.dtype)[1:].view(out.shape)
        got = torch.autograd.grad(out, leaf, grad)[0]
        _check_gradient(got, indices, grad.reshape(-1, table.shape[1]), 50, 0.5, 'bf16' if table.dtype == torch.bfloat16 else 'f32')


def test_broadcast_upstream_gradients():
    import efgs
    indices = torch.randint(0, 30, (1000,), device=DEVICE)
    table = torch.randn(30, 7, device=DEVICE, requires_grad=True)
    got = torch.autograd.grad(efgs.embedding(indices, table, 2.0).sum(), table)[0]
    want = 2.0 * torch.bincount(indices, minlength=30).float()[:, None].expand(30, 7)
    assert torch.equal(got, want)   # (whole numbers: exact)


def test_padding_row():
    import efgs
    indices, table, grad = _inputs(2000, 40, 6, 'f32', invalid=0.0)
    for padding in (0, 5, 39, -1, -40):
        out = efgs.embedding(indices, table, 1.0, padding)
        assert torch.equal(out, _plain(indices, table, 1.0))
        got = torch.autograd.grad(out, table, grad)[0]
        _check_gradient(got, indices, grad, 40, 1.0, 'f32', padding % 40)
    for padding in (40, -41):
        with pytest.raises(ValueError, match='padding_idx'):
            efgs.embedding(indices, table, 1.0, padding)


@pytest.mark.parametrize('rows', [50, 5000])
def test_odd_values_stay_in_their_rows(rows):
    """Infinities and NaN in a row of the table or upstream reach that row alone; those behind an index that counts nowhere reach none."""
    import efgs
    indices = torch.randint(2, rows, (3000,), device=DEVICE)
    indices[7], indices[8], indices[9] = 0, -3, 1
    table = torch.randn(rows, 8, device=DEVICE)
    table[0] = float('nan')
    leaf = table.requires_grad_()
    out = efgs.embedding(indices, leaf, 1.0, 1)
    assert bool(out[7].isnan().all()) and torch.equal(out[8], torch.zeros(8, device=DEVICE))
    grad = torch.randn(3000, 8, device=DEVICE)
    grad[7], grad[8], grad[9] = float('inf'), float('nan'), float('nan')
    got = torch.autograd.grad(out, leaf, grad)[0]
    assert bool((got[0] == float('inf')).all()) and torch.equal(got[1], torch.zeros(8, device=DEVICE))
    assert bool(got[2:].isfinite().all())


@pytest.mark.parametrize('n, rows, columns', [(200_000, 700, 24), (200_000, 7000, 24), (1_100_000, 4000, 8), (7000, 50_000, 8)])
def test_results_repeat_bit_for_bit(n, rows, columns):
    import efgs
    indices, table, grad = _inputs(n, rows, columns, 'f32')
    first = torch.autograd.grad(efgs.embedding(indices, table), table, grad)[0]
    for _ in range(3):
        assert torch.equal(first, torch.autograd.grad(efgs.embedding(indices, table), table, grad)[0])


def test_gradient_against_differences():
    """The lookup is linear in the table: differences of a weighted sum, in steps of 1/4 of small whole numbers, are exact."""
    import efgs
    indices = torch.tensor([3, 1, 3, -1, 0, 3], device=DEVICE)
    weight = torch.tensor(np.random.default_rng(0).integers(-4, 5, (6, 5)), device=DEVICE).float()
    table = torch.tensor(np.random.default_rng(1).integers(-4, 5, (4, 5)), device=DEVICE).float().requires_grad_()
    got = torch.autograd.grad((efgs.embedding(indices, table, 2.0) * weight).sum(), table)[0]
    with torch.no_grad():
        for r in range(4):
            for c in range(5):
                step = torch.zeros(4, 5, device=DEVICE)
                step[r, c] = 0.25
                ends = [(efgs.embedding(indices, table + s * step, 2.0) * weight).sum() for s in (1, -1)]
                assert float(ends[0] - ends[1]) / 0.5 == float(got[r, c])


def test_autograd_rules():
    import efgs
    indices = torch.randint(0, 9, (64,), device=DEVICE)
    table = torch.randn(9, 4, device=DEVICE, requires_grad=True)
    with torch.no_grad():
        assert not efgs.embedding(indices, table).requires_grad
    assert not efgs.embedding(indices, table.detach()).requires_grad
    out = efgs.embedding(indices, table)
    first = torch.autograd.grad(out.sum(), table, retain_graph=True)[0]
    assert torch.equal(first, torch.autograd.grad(out.sum(), table)[0])
    out = efgs.embedding(indices, table)
    upstream = torch.ones_like(out, requires_grad=True)
    again = torch.autograd.grad(out, table, upstream, create_graph=True)[0]
    with pytest.raises(RuntimeError, match='once_differentiable'):
        again.sum().backward()
    out = efgs.embedding(indices, table)
    indices[0] = (indices[0] + 1) % 9
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        out.sum().backward()


def test_on_a_stream_of_its_own():
    import efgs
    indices, table, grad = _inputs(100_000, 400, 16, 'f32')
    want = torch.autograd.grad(efgs.embedding(indices, table), table, grad)[0]
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        x = torch.ones(2048, 2048, device=DEVICE)
        for _ in range(8):
            x = x @ x * 1e-4
        moved = indices + (x[0, 0] * 0).long()
        got = torch.autograd.grad(efgs.embedding(moved, table), table, grad)[0]
    torch.cuda.current_stream().wait_stream(stream)
    assert torch.equal(got, want)


@pytest.mark.parametrize('rows', [500, 9000])
def test_graph_replays_match_eager(rows):
    """Lookup and gradient captured as one graph; every replay, on new values, equals the eager results."""
    import efgs
    indices, table, grad = _inputs(60_000, rows, 8, 'f32')
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            torch.autograd.grad(efgs.embedding(indices, table, 2.0), table, grad)
    torch.cuda.current_stream().wait_stream(side)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = efgs.embedding(indices, table, 2.0)
        got = torch.autograd.grad(out, table, grad)[0]
    for seed in range(4):
        new = _inputs(60_000, rows, 8, 'f32', seed=seed + 1)
        with torch.no_grad():
            indices.copy_(new[0])
            table.copy_(new[1])
            grad.copy_(new[2])
        leaf = table.detach().clone().requires_grad_()
        want = efgs.embedding(indices, leaf, 2.0)
        want_grad = torch.autograd.grad(want, leaf, grad)[0]
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want) and torch.equal(got, want_grad)


def test_outputs_past_2_to_the_32_elements():
    """1,050,000 rows of 4,100 (8.6 GB out, as much upstream): looked-up rows and gradients at both ends."""
    import efgs
    n, rows, columns = 1_050_000, 13, 4100
    assert n * columns > 1 << 32
    print('case embedding past 2^32', flush=True)
    table = torch.randn(rows, columns, device=DEVICE).bfloat16().requires_grad_()
    indices = torch.full((n,), 4, device=DEVICE)
    indices[-5:] = torch.arange(5, 10, device=DEVICE)
    indices[:5] = torch.tensor([10, 11, 12, 0, 1], device=DEVICE)
    out = efgs.embedding(indices, table, 3.0)
    for part in (slice(0, 10), slice(n - 10, n)):
        assert torch.equal(out[part], _plain(indices[part], table, 3.0))
    grad = torch.zeros(n, columns, dtype=torch.bfloat16, device=DEVICE)
    grad[-9:] = torch.randn(9, columns, device=DEVICE).bfloat16()
    grad[:9] = torch.randn(9, columns, device=DEVICE).bfloat16()
    got = torch.autograd.grad(out, table, grad)[0]
    ends = torch.cat([torch.arange(9), torch.arange(n - 9, n)]).to(DEVICE)
    _check_gradient(got, indices[ends], grad[ends], rows, 3.0, 'bf16')
