"""efgs.linear_cross_entropy on the GPU against the 64-bit oracle (oracle/training_ref.py).

Bars, e = 2^-24, u = half a step of the inputs' type relative to the value (2^-24, 2^-8, 2^-11): a logit is a float32 sum of D exact or
once-rounded products, off by dz <= 2 (D + 4) e scale sum |x w|, the 2 for matrix instructions that may cut where they align, and the product with
scale log2 e and its rounding 3 e |z|. A sum of exponentials of V table rows goes through at most 64 + V / 16 additions in a row, each exponential 4 e
off; so a loss is off by 2 max dz + (80 + V / 16) e + 4 e (|lse| + |z|), and a probability by that relative to it. g = weight (p - onehot) is rounded to the
type (u |g|, and 2^-38 for float16, whose g is held times 2^15), a gradient is a float32 sum of K values (at most 2 (K + 4) e of their magnitudes), scaled, and
rounded to the type: u of the value, float16 half its least step, 2^-25. Floats as three bfloat16 parts lose 2^-26 each and 2^-25 by the pairs left out, within the 4 beside D.
"""
import numpy as np
import pytest
import torch

import training_ref as R

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = {'f32': (torch.float32, E, 0.0, 0.0), 'bf16': (torch.bfloat16, 2.0 ** -8, 0.0, 0.0), 'f16': (torch.float16, 2.0 ** -11, 2.0 ** -25, 2.0 ** -38)}
DEVICE = 'cuda:0'


def inputs(n, rows, columns, dtype, seed=0, left_out=0.1, index=torch.int64, sharp=8.0, scale=1.0):
    rng = np.random.default_rng(seed)
    kind = TYPES[dtype][0]
    table = torch.tensor(rng.normal(size=(rows, columns)) * 2.0 / (scale * np.sqrt(columns)), device=DEVICE).to(kind)
    targets = rng.integers(0, rows, n)
    pull = torch.tensor(rng.random((n, 1)) * sharp * scale / 4.0, device=DEVICE)
    features = (torch.tensor(rng.normal(size=(n, columns)), device=DEVICE) + pull * table[torch.tensor(targets, device=DEVICE)].double()).to(kind)
    wrong = np.array([-1, -100, rows, rows + 7, -(1 << 31), (1 << 31) - 1])
    pick = rng.random(n) < left_out
    targets[pick] = wrong[rng.integers(0, 6, int(pick.sum()))]
    return features, table, torch.tensor(targets, device=DEVICE).to(index), torch.tensor(rng.normal(size=n), dtype=torch.float32, device=DEVICE)


def bounds(features, table, targets, weights, scale, dtype, gradient=True):
    """(losses and their bars, gradients and their bars) as numpy arrays."""
    _, u, least, held = TYPES[dtype]
    x, w = features.detach().double().cpu().numpy(), table.detach().double().cpu().numpy()
    y = targets.cpu().numpy()
    weights = np.asarray(weights, np.float64)
    inside = (y >= 0) & (y < len(w))
    x = np.where(inside[:, None], x, 0.0)
    losses, p, g, dx, dw = R.cross_entropy(x, w, y, scale, weights)
    size, z = abs(scale) * (np.abs(x) @ np.abs(w).T), scale * (x @ w.T)
    dz = 2 * (x.shape[1] + 4) * E * size + 3 * E * np.abs(z)
    off = 2 * dz.max(1) + (80 + len(w) / 16) * E + 8 * E * (np.abs(z).max(1) + np.log(len(w)) + 1)
    loss_bar = np.where(inside, off, 0.0)
    if not gradient:
        return losses, loss_bar
    dg = np.abs(weights)[:, None] * (p * off[:, None] * 1.01 + 2 * E) * inside[:, None] + u * np.abs(g) * 1.02 + held * np.abs(weights).max(initial=1.0)
    dg *= inside[:, None]
    aw, ax, ag, s = np.abs(w), np.abs(x), np.abs(g) + dg, abs(scale)
    bar_x = s * (dg @ aw + 2 * (len(w) + 4) * E * (ag @ aw)) * (1 + 4 * E)
    bar_w = s * (dg.T @ ax + 2 * (len(x) + 4) * E * (ag.T @ ax)) * (1 + 4 * E)
    bar_x += u * (np.abs(dx) + bar_x) + least
    bar_w += u * (np.abs(dw) + bar_w) + least
    return losses, loss_bar, dx, bar_x, dw, bar_w


def within(name, got, want, bar):
    got = got.detach().double().cpu().numpy()
    off = np.abs(got - want)
    assert got.shape == want.shape and np.all(off <= bar), (name, float(np.max(off / np.maximum(bar, 1e-300))), np.unravel_index(np.argmax(off - bar), off.shape))


def check(n, rows, columns, dtype, scale=1.0, reduction='mean', grads=(True, True), **how):
    import efgs
    print(f'case cross entropy n={n} rows={rows} columns={columns} {dtype} {reduction} {how}', flush=True)
    features, table, targets, upstream = inputs(n, rows, columns, dtype, scale=scale, **how)
    features.requires_grad_(grads[0])
    table.requires_grad_(grads[1])
    inside = int(((targets >= 0) & (targets < rows)).sum())
    if reduction == 'none':
        weights, up = upstream.double().cpu().numpy(), upstream
    else:
        up = upstream[0] if n else torch.tensor(0.7, device=DEVICE)
        weights = np.full(n, float(up) / (max(inside, 1) if reduction == 'mean' else 1))
    losses, loss_bar, dx, bar_x, dw, bar_w = bounds(features, table, targets, weights, scale, dtype)
    loss = efgs.linear_cross_entropy(features, table, targets, scale, reduction)
    with torch.no_grad():
        alone = efgs.linear_cross_entropy(features, table, targets, scale, reduction)
    for value in (loss, alone):  # (without a gradient a few rows take another way)
        assert value.dtype == torch.float32
        if reduction == 'none':
            within('losses', value, losses, loss_bar)
            assert np.all(value.detach().cpu().numpy()[loss_bar == 0] == 0)
        else:
            share = max(inside, 1) if reduction == 'mean' else 1
            within('loss', value, np.asarray(losses.sum() / share), np.asarray((loss_bar.sum() + 2 * E * losses.sum()) / share + 1e-300))
    loss.backward(up)
    if grads[0]:
        assert features.grad.dtype == features.dtype
        within('features', features.grad, dx, bar_x)
    else:
        assert features.grad is None
    if grads[1]:
        within('table', table.grad, dw, bar_w)
    else:
        assert table.grad is None
    return features, table, targets, up, loss


COLUMNS = [1, 3, 8, 15, 16, 33, 45, 64, 65, 72, 128, 136, 200, 257, 333, 512]


@pytest.mark.parametrize('columns', COLUMNS)
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_widths(columns, dtype):
    check(301, 1003, columns, dtype, seed=columns)


@pytest.mark.parametrize('n', [1, 2, 15, 16, 17, 64, 65, 255, 256, 257, 1025])
@pytest.mark.parametrize('columns,dtype', [(8, 'f32'), (96, 'bf16'), (200, 'f32'), (130, 'f16')])
def test_row_counts(n, columns, dtype):
    check(n, 517, columns, dtype, seed=n, reduction='none')


@pytest.mark.parametrize('rows', [1, 2, 15, 16, 17, 127, 128, 129, 255, 256, 257, 2049, 5003])
@pytest.mark.parametrize('columns,dtype', [(8, 'f32'), (64, 'bf16'), (300, 'f16')])
def test_table_sizes(rows, columns, dtype):
    check(133, rows, columns, dtype, seed=rows, reduction='sum')


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('scale', [0.25, -1.5, 10.0])
def test_reductions_and_scales(dtype, reduction, scale):
    check(260, 700, 72, dtype, scale=scale, reduction=reduction, index=torch.int32)


@pytest.mark.parametrize('grads', [(True, False), (False, True)])
@pytest.mark.parametrize('dtype,columns', [('f32', 8), ('f32', 150), ('bf16', 256)])
def test_one_gradient_alone(dtype, columns, grads):
    check(100, 400, columns, dtype, grads=grads)


@pytest.mark.parametrize('dtype,columns', [('f32', 8), ('f32', 150), ('bf16', 8), ('bf16', 256), ('f16', 77)])
@pytest.mark.parametrize('left_out', [0.0, 0.9, 1.0])
def test_rows_left_out(dtype, columns, left_out):
    for reduction in ('mean', 'none'):
        f, t, targets, up, loss = check(600, 300, columns, dtype, left_out=left_out, reduction=reduction)
        out = (targets < 0) | (targets >= 300)
        assert torch.all(f.grad[out] == 0)
        if left_out == 1.0:
            assert torch.all(loss == 0) and torch.all(t.grad == 0)


@pytest.mark.parametrize('dtype,columns', [('f32', 8), ('f32', 150), ('bf16', 8), ('bf16', 256), ('f16', 77)])
def test_what_stands_in_rows_left_out_reaches_nothing(dtype, columns):
    import efgs
    features, table, targets, upstream = inputs(300, 500, columns, dtype, seed=3, left_out=0.3)
    out = (targets < 0) | (targets >= 500)
    assert int(out.sum()) > 10
    results = []
    for value in (0.0, float('nan'), float('inf'), -float('inf')):
        x, w, up = features.clone(), table.clone().requires_grad_(), upstream.clone()
        x[out] = value
        up[out] = value
        x.requires_grad_()
        loss = efgs.linear_cross_entropy(x, w, targets, reduction='none')
        loss.backward(up)
        results.append((loss.detach(), x.grad, w.grad))
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)


@pytest.mark.parametrize('n,rows,columns', [(0, 5, 4), (4, 0, 4), (4, 5, 0), (0, 0, 3), (0, 5, 200)])
@pytest.mark.parametrize('reduction', ['mean', 'sum', 'none'])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_empty_sides(n, rows, columns, reduction, dtype):
    import efgs
    x, w = (torch.randn(k, columns, device=DEVICE, dtype=TYPES[dtype][0], requires_grad=True) for k in (n, rows))
    y = torch.zeros(n, dtype=torch.int64, device=DEVICE)
    loss = efgs.linear_cross_entropy(x, w, y, reduction=reduction)
    counted = n if rows else 0   # (rows that count have no columns here: equal logits)
    each = np.full(n, np.log(rows) if rows else 0.0)
    want = each if reduction == 'none' else each.sum() / (max(counted, 1) if reduction == 'mean' else 1)
    assert np.allclose(loss.detach().cpu().numpy(), want, atol=1e-6)
    loss.sum().backward()
    assert x.grad.shape == x.shape and w.grad.shape == w.shape and torch.all(x.grad == 0) and torch.all(w.grad == 0)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('columns', [16, 136])
def test_shapes_strides_and_alignment(dtype, columns):
    """Leading dimensions, transposed and offset views: the same bits as of contiguous copies."""
    import efgs
    kind = TYPES[dtype][0]
    rng = torch.Generator(DEVICE).manual_seed(5)
    base = torch.randn(3, columns + 3, 40, generator=rng, device=DEVICE).to(kind)
    wide = torch.randn(301, columns + 5, generator=rng, device=DEVICE).to(kind)
    targets = torch.randint(-1, 300, (40, 3), generator=rng, device=DEVICE).t()
    for x, w in ((base[:, 1:columns + 1].transpose(1, 2), wide[1:, 3:columns + 3]), (base[:, 1:columns + 1].transpose(1, 2), wide[1:, :columns].t().contiguous().t())):
        results = []
        for a, b, y in ((x, w, targets), (x.contiguous(), w.contiguous(), targets.contiguous())):
            a, b = a.detach().requires_grad_(), b.detach().requires_grad_()
            loss = efgs.linear_cross_entropy(a, b, y, reduction='none')
            assert loss.shape == (3, 40)
            results.append((loss.detach(), *torch.autograd.grad(loss, (a, b), torch.ones_like(loss))))
        for a, b in zip(*results):
            assert torch.equal(a, b)


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_far_logits(dtype):
    """Logits of hundreds, equal ones, and a target that no probability is left for."""
    import efgs
    x = torch.zeros(4, 80, device=DEVICE)
    x[0, 0], x[1, 0], x[2, 1] = 30.0, -30.0, 30.0
    w = torch.zeros(50, 80, device=DEVICE)
    w[:, 0] = torch.linspace(-16, 16, 50, device=DEVICE).to(TYPES[dtype][0]).float()
    y = torch.tensor([0, 0, 7, 49], device=DEVICE)
    x, w = x.to(TYPES[dtype][0]).requires_grad_(), w.to(TYPES[dtype][0]).requires_grad_()
    loss = efgs.linear_cross_entropy(x, w, y, reduction='none')
    losses, bar, dx, bar_x, dw, bar_w = bounds(x, w, y, np.ones(4), 1.0, dtype)
    within('losses', loss, losses, bar)
    loss.sum().backward()
    within('features', x.grad, dx, bar_x)
    within('table', w.grad, dw, bar_w)


@pytest.mark.parametrize('dtype,columns', [('f32', 8), ('f32', 150), ('bf16', 8), ('bf16', 256), ('f16', 256)])
def test_infinities_and_nan_are_passed_on(dtype, columns):
    import efgs
    features, table, targets, _ = inputs(70, 300, columns, dtype, left_out=0.0)
    features[3, 0] = float('nan')
    features.requires_grad_()
    loss = efgs.linear_cross_entropy(features, table, targets, reduction='none')
    assert bool(torch.isnan(loss[3])) and int(torch.isnan(loss).sum()) == 1
    loss.sum().backward()
    assert torch.all(torch.isnan(features.grad[3])) and int(torch.isnan(features.grad).any(1).sum()) == 1


@pytest.mark.parametrize('dtype,columns', [('f32', 8), ('f32', 150), ('bf16', 16), ('bf16', 256), ('f16', 256)])
def test_the_same_bits_every_time(dtype, columns):
    import efgs
    features, table, targets, upstream = inputs(777, 3001, columns, dtype)
    features.requires_grad_()
    table.requires_grad_()
    first = None
    for _ in range(3):
        loss = efgs.linear_cross_entropy(features, table, targets, reduction='none')
        now = (loss.detach(), *torch.autograd.grad(loss, (features, table), upstream))
        first = first or now
        for a, b in zip(first, now):
            assert torch.equal(a, b)


@pytest.mark.parametrize('dtype,columns', [('f32', 8), ('f32', 150), ('bf16', 256)])
def test_a_captured_step_replays(dtype, columns):
    import efgs
    features, table, targets, _ = inputs(300, 1000, columns, dtype)
    features.requires_grad_()
    table.requires_grad_()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            efgs.linear_cross_entropy(features, table, targets).backward()
            features.grad = table.grad = None
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        loss = efgs.linear_cross_entropy(features, table, targets)
        loss.backward()
    held = (features.grad, table.grad)
    for seed in range(4):
        other = inputs(300, 1000, columns, dtype, seed=seed + 10, left_out=0.2 * seed)
        with torch.no_grad():
            features.copy_(other[0])
            table.copy_(other[1])
            targets.copy_(other[2])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in (loss.detach(), *held)]
        a, b = features.detach().clone().requires_grad_(), table.detach().clone().requires_grad_()
        eager = efgs.linear_cross_entropy(a, b, targets)
        eager.backward()
        for x, y in zip(got, (eager.detach(), a.grad, b.grad)):
            assert torch.equal(x, y)


def test_two_calls_on_two_streams():
    import efgs
    work = [inputs(500, 2000, c, d, seed=k) for k, (c, d) in enumerate(((8, 'f32'), (256, 'bf16'), (150, 'f32'), (128, 'f16')))]
    def step(features, table, targets, upstream):
        a, b = features.detach().requires_grad_(), table.detach().requires_grad_()
        loss = efgs.linear_cross_entropy(a, b, targets, reduction='none')
        return (loss.detach(), *torch.autograd.grad(loss, (a, b), upstream))
    alone = [step(*w) for w in work]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in work]
    together = []
    for s, w in zip(streams, work):
        with torch.cuda.stream(s):
            together.append(step(*w))
    torch.cuda.synchronize()
    for a, b in zip(alone, together):
        for x, y in zip(a, b):
            assert torch.equal(x, y)


def test_an_in_place_change_of_the_table_is_refused_and_of_the_features_does_not_matter():
    import efgs
    features, table, targets, _ = inputs(50, 100, 16, 'f32')
    x, w = features.clone().requires_grad_(), table.clone().requires_grad_()
    want = torch.autograd.grad(efgs.linear_cross_entropy(x, w, targets), (x, w))
    y = x * 1.0
    loss = efgs.linear_cross_entropy(y, w, targets)
    with torch.no_grad():
        y.zero_()
    got = torch.autograd.grad(loss, (y, w), retain_graph=True)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    with torch.no_grad():
        w.zero_()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        torch.autograd.grad(loss, (y, w))


def test_second_derivatives_raise():
    import efgs
    features, table, targets, _ = inputs(20, 30, 16, 'f32')
    features.requires_grad_()
    up = torch.ones((), device=DEVICE, requires_grad=True)
    grad = torch.autograd.grad(efgs.linear_cross_entropy(features, table, targets), features, up, create_graph=True)[0]
    with pytest.raises(RuntimeError, match='once_differentiable'):
        torch.autograd.grad(grad.sum(), up)


@pytest.mark.parametrize('n', [1, 2, 3, 16, 17, 32, 33, 63, 64, 65])
@pytest.mark.parametrize('columns', [1, 5, 31, 32, 33, 63, 64, 65, 127, 129, 200, 1000, 1024])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_a_few_rows_without_a_gradient(n, columns, dtype):
    import efgs
    rows = 37 * n + columns % 97 + 1
    features, table, targets, _ = inputs(n, rows, columns, dtype, seed=n + columns, left_out=0.2)
    losses, bar = bounds(features, table, targets, np.ones(n), 0.8, dtype, gradient=False)
    within('losses', efgs.linear_cross_entropy(features, table, targets, 0.8, 'none'), losses, bar)
    count = max(1, int(((targets >= 0) & (targets < rows)).sum()))
    mean = efgs.linear_cross_entropy(features, table, targets, 0.8)
    within('mean', mean, np.asarray(losses.sum() / count), np.asarray((bar.sum() + 2 * E * losses.sum()) / count + 1e-300))
    odd = torch.empty(rows * (columns + 3) + 1, dtype=table.dtype, device=DEVICE)[1:].view(rows, columns + 3)[:, 2:columns + 2]
    odd.copy_(table)
    assert torch.equal(efgs.linear_cross_entropy(features, odd, targets, 0.8), mean)


def test_what_stands_in_few_rows_left_out_reaches_nothing():
    import efgs
    features, table, targets, _ = inputs(40, 500, 100, 'bf16', left_out=0.3)
    out = (targets < 0) | (targets >= 500)
    results = []
    for value in (0.0, float('nan'), float('inf')):
        x = features.clone()
        x[out] = value
        results.append((efgs.linear_cross_entropy(x, table, targets, reduction='none'), efgs.linear_cross_entropy(x, table, targets)))
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)
    features[3] = float('nan')
    targets[3] = 1
    assert bool(torch.isnan(efgs.linear_cross_entropy(features, table, targets, reduction='none')[3]))


def test_pieces_and_lists_of_many_rows():
    """More rows than a block counts by itself, more of the table than a piece holds."""
    check(20_001, 600, 8, 'f32', seed=9)
    check(17_000, 300, 130, 'f32', seed=9, reduction='none')
    check(17_000, 300, 64, 'bf16', seed=10)


@pytest.mark.parametrize('n,train', [(3, False), (300, False), (70, True)])
def test_offsets_past_32_bits(n, train):
    """A table of more than 4 GB: its last rows are met, and get their gradients."""
    import efgs
    rows, columns = 1_200_003, 2048
    table = torch.zeros(rows, columns, dtype=torch.bfloat16, device=DEVICE)
    rng = torch.Generator(DEVICE).manual_seed(1)
    special = torch.tensor([0, 1, 524_287, 1_048_576, 1_048_577, rows - 2, rows - 1], device=DEVICE)
    table[special] = (torch.randn(len(special), columns, generator=rng, device=DEVICE) / 32).bfloat16()
    x = torch.randn(n, columns, generator=rng, device=DEVICE).bfloat16()
    targets = special[torch.arange(n, device=DEVICE) % len(special)]
    z = x.double() @ table[special].double().t()
    total = torch.log(torch.exp(z).sum(1) + (rows - len(special)))
    at = torch.arange(n, device=DEVICE) % len(special)
    want = total - z[torch.arange(n, device=DEVICE), at]
    if train:
        table.requires_grad_()
        x.requires_grad_()
    loss = efgs.linear_cross_entropy(x, table, targets, reduction='none')
    # (float32 logits of 2,048 products and 1.2 million exponentials: far inside of 1e-3)
    assert torch.all((loss.detach().double() - want).abs() < 1e-3)
    if train:
        loss.sum().backward()
        g = torch.exp(z - total[:, None])
        g[torch.arange(n, device=DEVICE), at] -= 1.0
        for got, exact in ((table.grad[special].double(), g.t() @ x.detach().double()), (x.grad.double(), g @ table.detach()[special].double())):
            # (bfloat16 logits' gradients and one rounding: 2^-8 each of sums of 70 and 7 terms)
            assert float((got - exact).abs().max()) <= 2.0 ** -6 * float(exact.abs().max())
        rest = table.grad[2].double()
        assert torch.all(torch.isfinite(rest)) and float(rest.abs().max()) < 1e-3


def test_a_graph_kept_and_run_twice():
    import efgs
    features, table, targets, upstream = inputs(200, 300, 96, 'bf16')
    features.requires_grad_()
    table.requires_grad_()
    loss = efgs.linear_cross_entropy(features, table, targets, reduction='none')
    first = torch.autograd.grad(loss, (features, table), upstream, retain_graph=True)
    second = torch.autograd.grad(loss, (features, table), upstream)
    for a, b in zip(first, second):
        assert torch.equal(a, b)


@pytest.mark.parametrize('columns', [8, 96])
def test_all_rows_of_one_target(columns):
    """Every packed row's own target in one tile of the table, more of them than are listed at once."""
    import efgs
    n = 10_000
    rng = torch.Generator(DEVICE).manual_seed(3)
    x = torch.randn(n, columns, generator=rng, device=DEVICE).bfloat16().requires_grad_()
    w = (torch.randn(600, columns, generator=rng, device=DEVICE) / 8).bfloat16().requires_grad_()
    y = torch.full((n,), 333, device=DEVICE)
    efgs.linear_cross_entropy(x, w, y, reduction='sum').backward()
    _, _, g, dx, dw = R.cross_entropy(x.detach().double().cpu().numpy(), w.detach().double().cpu().numpy(), y.cpu().numpy(), 1.0, np.ones(n))
    losses, _, dx, bar_x, dw, bar_w = bounds(x, w, y, np.ones(n), 1.0, 'bf16')
    within('features', x.grad, dx, bar_x)
    within('table', w.grad, dw, bar_w)
    # the target's row itself: without its residuals the 10,000 roundings of about -1 would be most of its error
    off = np.abs(w.grad.double().cpu().numpy()[333] - dw[333])
    assert np.all(off <= 2.0 ** -8 * np.abs(dw[333]) * 1.01 + 2.0 ** -15 * (np.abs(g[:, 333]) @ np.abs(x.detach().double().cpu().numpy())))


def test_saved_tensors_may_be_packed_by_hooks():
    import efgs
    features, table, targets, _ = inputs(100, 200, 64, 'f32')
    features.requires_grad_()
    table.requires_grad_()
    want = torch.autograd.grad(efgs.linear_cross_entropy(features, table, targets), (features, table))
    with torch.autograd.graph.save_on_cpu():
        loss = efgs.linear_cross_entropy(features, table, targets)
    for a, b in zip(want, torch.autograd.grad(loss, (features, table))):
        assert torch.equal(a, b)


@pytest.mark.parametrize('columns', [32, 96])
def test_an_infinite_gradient_of_one_row_leaves_the_others_theirs(columns):
    """float16 gradients of the size a loss scale makes them, one overflowed to infinity: only its own row (and the table, which it has a part in) loses them."""
    import efgs
    features, table, targets, upstream = inputs(90, 300, columns, 'f16', left_out=0.0)
    features.requires_grad_()
    upstream = upstream * 1000.0
    upstream[17] = float('inf')
    grad, = torch.autograd.grad(efgs.linear_cross_entropy(features, table, targets, reduction='none'), features, upstream)
    assert not bool(torch.isfinite(grad[17]).any())
    weights = upstream.double().cpu().numpy()
    weights[17] = 0.0
    _, _, dx, bar_x, _, _ = bounds(features, table, targets, weights, 1.0, 'f16')
    dx[17] = bar_x[17] = 0.0
    grad[17] = 0.0
    within('features', grad, dx, bar_x)


@pytest.mark.parametrize('dtype,columns', [('f32', 24), ('f32', 96), ('bf16', 24), ('bf16', 96), ('f16', 136)])
@pytest.mark.parametrize('n', [5, 150])
def test_broadcast_rows_and_shared_tensors(dtype, columns, n):
    """One feature row for all targets, one table row for all codes, and one tensor as both, with 32-bit targets: as of their copies."""
    import efgs
    rng = torch.Generator(DEVICE).manual_seed(9)
    kind = TYPES[dtype][0]
    rows = torch.randn(150, columns, generator=rng, device=DEVICE).to(kind)
    one = torch.randn(1, columns, generator=rng, device=DEVICE).to(kind)
    y = torch.randint(-1, 150, (n,), generator=rng, device=DEVICE, dtype=torch.int32)

    def run(x, w, grads):
        loss = efgs.linear_cross_entropy(x, w, y, 0.3)
        with torch.no_grad():
            alone = efgs.linear_cross_entropy(x, w, y, 0.3)
        return loss.detach(), alone, *torch.autograd.grad(loss, grads)

    for x, w in ((one.expand(n, columns), rows), (rows[:n], one.expand(150, columns))):
        a, b = x.detach().requires_grad_(), w.detach().requires_grad_()
        c, d = x.contiguous().requires_grad_(), w.contiguous().requires_grad_()
        for got, want in zip(run(a, b, (a, b)), run(c, d, (c, d))):
            assert torch.equal(got, want)
    x, w = rows[:n].clone().requires_grad_(), rows.clone().requires_grad_()
    both = rows.clone().requires_grad_()
    loss, alone, dx, dw = run(x, w, (x, w))
    got, got_alone, grad = run(both[:n], both, (both,))
    assert torch.equal(got, loss) and torch.equal(got_alone, alone)
    want = dw.clone()
    want[:n] += dx
    assert torch.equal(grad, want)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_rows_of_millions_of_columns(dtype):
    """All but seven columns zero: as those columns alone."""
    import efgs
    columns, kind = (1 << 21) + 72, TYPES[dtype][0]
    at = torch.tensor([0, 1, 63, 1 << 20, (1 << 21) - 1, 1 << 21, columns - 1], device=DEVICE)
    rng = torch.Generator(DEVICE).manual_seed(4)
    x, w = (torch.randn(k, 7, generator=rng, device=DEVICE).to(kind).requires_grad_() for k in (3, 5))
    y = torch.tensor([4, -1, 2], device=DEVICE)
    want = efgs.linear_cross_entropy(x, w, y, reduction='none')
    want_x, want_w = torch.autograd.grad(want, (x, w), torch.ones_like(want))
    wide_x, wide_w = (torch.zeros(len(t), columns, device=DEVICE, dtype=kind).index_copy_(1, at, t.detach()).requires_grad_() for t in (x, w))
    loss = efgs.linear_cross_entropy(wide_x, wide_w, y, reduction='none')
    grad_x, grad_w = torch.autograd.grad(loss, (wide_x, wide_w), torch.ones_like(loss))
    # (logits of seven products of at most about 9; bf16: both ways round g and the result)
    u = TYPES[dtype][1]
    assert torch.all((loss - want).abs() <= 2.0 ** -18)
    for got, value in ((grad_x, want_x), (grad_w, want_w)):
        assert int((got != 0).sum()) == int((got[:, at] != 0).sum())
        assert torch.all((got[:, at].float() - value.float()).abs() <= 4 * u * (value.float().abs() + 3.0 * 5) + 2.0 ** -16)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_more_rows_of_one_target_than_a_list_holds(dtype):
    """Rows of one column each, all of one target, so many that a block looks them up in several parts: every one counts once. With n_c rows of column c and
    p_c the softmax of the table's column, the table's gradient is n_c (p_c - onehot) and a row's the sum of (p_c - onehot) w.

    Logits are single products (exact but for 2^-25), a sum of 4,096 exponentials is (64 + 4096 / 16) e off at most, so a probability by 2^-15 of it; the at
    most five rows of a column add up exactly but for their roundings; a row's gradient is a float32 sum of at most 6 * 4096 / 32 steps, 2^-13 of its terms."""
    import efgs
    n, rows, columns, target = 20_000, 4_096, 4_096, 333
    kind, u, _, _ = TYPES[dtype]
    rng = torch.Generator(DEVICE).manual_seed(6)
    column = torch.arange(n, device=DEVICE) % columns
    x = torch.zeros(n, columns, device=DEVICE, dtype=kind).scatter_(1, column[:, None], 1.0).requires_grad_()
    w = torch.randn(rows, columns, generator=rng, device=DEVICE).to(kind).requires_grad_()
    efgs.linear_cross_entropy(x, w, torch.full((n,), target, device=DEVICE), reduction='sum').backward()
    wide = w.detach().double()
    g = torch.softmax(wide, 0)
    p = g.clone()
    g[target] -= 1.0
    count = torch.bincount(column, minlength=columns)
    dw, size = count * g, count * p
    off = (w.grad.double() - dw).abs()
    assert torch.all(off <= 2.0 ** -14 * size + 2.0 * u * (count * g.abs()) + u * dw.abs()), float((off / (size + dw.abs())).max())
    some = torch.tensor([0, 1, 777, 4_095, 4_096, 8_191, 8_192, 16_384, n - 1], device=DEVICE)
    c = column[some]
    dx, size = g[:, c].t() @ wide, g[:, c].t().abs() @ wide.abs()
    off = (x.grad[some].double() - dx).abs()
    assert torch.all(off <= (2.0 ** -13 + 2.0 ** -14 + 2.0 * u) * size + u * dx.abs()), float((off / size).max())


@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('n,rows', [(6_399, 100), (6_400, 100), (6_464, 100), (9_001, 17), (700, 2)])
def test_many_rows_of_each_target(n, rows, dtype):
    """About where the targets' gradients are no longer added to the table's apart (64 rows of each), and past it."""
    check(n, rows, 136, dtype, reduction='none')


@pytest.mark.parametrize('dtype,columns', [('f32', 16), ('f32', 96), ('bf16', 96)])
@pytest.mark.parametrize('grads', [(True, False), (False, True), (True, True)])
def test_a_penalty_on_a_gradient_raises(dtype, columns, grads):
    """The gradients depend on features and table themselves: what is differentiated through them raises, also where the upstream gradient asks for none."""
    import efgs
    features, table, targets, _ = inputs(20, 30, columns, dtype)
    leaves = [t.requires_grad_() for t, wanted in zip((features, table), grads) if wanted]
    x = features * 1.0   # (not a leaf: its own graph is part of what is differentiated)
    loss = efgs.linear_cross_entropy(x, table, targets)
    want = torch.autograd.grad(efgs.linear_cross_entropy(x, table, targets), leaves, retain_graph=True)
    got = torch.autograd.grad(loss, leaves, create_graph=True)
    for a, b in zip(got, want):
        assert a.requires_grad and not b.requires_grad and torch.equal(a, b)
        for leaf in leaves:
            with pytest.raises(RuntimeError, match='once_differentiable'):
                torch.autograd.grad(loss.float() + a.float().pow(2).sum(), leaf, retain_graph=True)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        (loss + got[0].float().pow(2).sum()).backward()


@pytest.mark.parametrize('dtype,n,rows', [('bf16', 40_000, 520), ('bf16', 8_320, 130), ('bf16', 5_000, 520), ('f16', 270_000, 4_100)])
def test_roundings_that_are_all_alike(dtype, n, rows):
    """All rows of one target, many of them for each table row, and a table of zeros: every row's own gradient is 1 / rows - 1, which the type rounds the same
    way every time. The target's row of the table's gradient is still one rounding off.

    Features are 1, 2 or 3: the sum of p x is off by 2^-24 for each of its steps of 32 rows and a few more, (n / 32 + 64) e of its size, twice for what the matrix
    instruction may cut; what a rounding lost, u of the whole, is itself held to u of it; then half a step of the result."""
    import efgs
    kind, u, _, _ = TYPES[dtype]
    rng = torch.Generator(DEVICE).manual_seed(n)
    columns, target = 96, 77
    x = torch.randint(1, 4, (n, columns), generator=rng, device=DEVICE).to(kind)
    w = torch.zeros(rows, columns, device=DEVICE, dtype=kind, requires_grad=True)
    efgs.linear_cross_entropy(x, w, torch.full((n,), target, device=DEVICE)).backward()
    dw = (1.0 / rows - 1.0) * x.double().mean(0)
    off = (w.grad[target].double() - dw).abs()
    inner = dw.abs() * (2 * (n / 32 + 64) * E + u * u)
    step = 2.0 ** torch.floor(torch.log2(dw.abs() + inner)) * 2 * u   # of the result
    assert torch.all(off <= step / 2 + inner), float((off / step).max())


def check_on_device(n, rows, columns, dtype, seed):
    """`check` with a weight for each row, oracle and bars in 64 bits on the GPU (the same formulas): sizes that would take long on the CPU."""
    import efgs
    print(f'case cross entropy on the device n={n} rows={rows} columns={columns} {dtype}', flush=True)
    _, u, least, held = TYPES[dtype]
    features, table, targets, weights = inputs(n, rows, columns, dtype, seed=seed)
    loss = efgs.linear_cross_entropy(features.requires_grad_(), table.requires_grad_(), targets, reduction='none')
    grad_x, grad_w = torch.autograd.grad(loss, (features, table), weights)
    inside = (targets >= 0) & (targets < rows)
    x, w = features.detach().double() * inside[:, None], table.detach().double()
    ax, aw, up, at = x.abs(), w.abs(), (weights.double() * inside)[:, None], inside.nonzero()[:, 0]
    z = x @ w.t()
    off = 2 * (2 * (columns + 4) * E * (ax @ aw.t()) + 3 * E * z.abs()).amax(1) + (80 + rows / 16) * E + 8 * E * (z.abs().amax(1) + np.log(rows) + 1)
    total = torch.logsumexp(z, 1)
    want = torch.zeros(n, dtype=torch.float64, device=DEVICE)
    want[at] = total[at] - z[at, targets[at].long()]
    assert torch.all((loss.detach().double() - want).abs() <= off * inside)
    g = torch.exp(z - total[:, None])
    del z
    dg = up.abs() * (g * off[:, None] * 1.01 + 2 * E)
    g[at, targets[at].long()] -= 1.0
    g *= up
    dg += (u * g.abs() * 1.02 + held * float(up.abs().max())) * inside[:, None]
    dx, dw = g @ w, g.t().contiguous() @ x
    ag = g.abs() + dg
    bar_x = (dg @ aw + 2 * (rows + 4) * E * (ag @ aw)) * (1 + 4 * E)
    bar_w = (dg.t().contiguous() @ ax + 2 * (n + 4) * E * (ag.t().contiguous() @ ax)) * (1 + 4 * E)
    for name, got, value, bar in (('features', grad_x, dx, bar_x), ('table', grad_w, dw, bar_w)):
        miss = (got.double() - value).abs() - (bar + u * (value.abs() + bar) + least)
        assert bool((miss <= 0).all()), (name, float(miss.max()), int(miss.argmax()) // columns)


@pytest.mark.parametrize('n,rows,columns,dtype', [
    (20_001, 7_001, 72, 'bf16'), (20_001, 7_001, 72, 'f16'), (20_001, 2_600, 72, 'f32'),      # two pieces
    (20_001, 13_001, 136, 'bf16'), (17_000, 17_009, 77, 'f16'), (20_001, 4_999, 65, 'f32'),   # three, tables that are copied
])
def test_several_pieces_of_the_table_the_last_one_shorter(n, rows, columns, dtype):
    """A piece's logits' gradients take 256 MB at most: for 20,001 rows 6,400 table rows of a 16-bit type, 2,048 of float32; the pieces are alike but for the
    last one."""
    check_on_device(n, rows, columns, dtype, seed=rows)


@pytest.mark.parametrize('columns', [32, 136])
def test_rows_of_small_weights_beside_large_ones(columns):
    """float16, weights from 1 down to 2^-20: every row's gradient as the formula has it, against bars that count each row's own weight but for the share of the
    largest one that float16 holds g to (2^-38)."""
    import efgs
    features, table, targets, _ = inputs(210, 700, columns, 'f16', left_out=0.0)
    features.requires_grad_()
    weights = 2.0 ** -(torch.arange(210, device=DEVICE) % 21).float()
    up = weights * 512.0
    grad, = torch.autograd.grad(efgs.linear_cross_entropy(features, table, targets, reduction='none'), features, up)
    _, _, dx, bar_x, _, _ = bounds(features, table, targets, up.double().cpu().numpy(), 1.0, 'f16')
    within('features', grad, dx, bar_x)
