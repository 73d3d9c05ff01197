"""efgs.balance_loss on the GPU against the 64-bit oracle (oracle/training_ref.py).

Bars, e = 2^-24, u half a step of the type relative to the value: z - max is off by e of it, its product with log2 e by 2 e |z| more, the exponential 2 e; a sum of
E of them goes through at most 40 additions in a row, and the quotient 2 e: a probability is off by r = (2 max |z - max| + 60) e of itself. Sums over rows go
through at most ceil(N / 1024) + 20 additions. The gradient p (share - mean) factor: mean off by (r + 45 e) of itself, then 4 e, then u, float16 half its least step.
"""
import numpy as np
import pytest
import torch

import training_ref as R

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = {'f32': (torch.float32, E, 0.0), 'bf16': (torch.bfloat16, 2.0 ** -8, 0.0), 'f16': (torch.float16, 2.0 ** -11, 2.0 ** -25)}
DEVICE = 'cuda:0'


def inputs(n, experts, chosen, dtype, seed=0, left_out=0.1, index=torch.int64, masked=0.0):
    rng = np.random.default_rng(seed)
    z = rng.normal(size=(n, experts)) * 2 + rng.normal(size=experts)
    if masked:
        z[rng.random((n, experts)) < masked] = -np.inf
    logits = torch.tensor(z, device=DEVICE).to(TYPES[dtype][0])
    indices = rng.integers(0, experts, (n, chosen))
    wrong = np.array([-1, experts, experts + 9, -(1 << 31), (1 << 31) - 1])
    pick = rng.random(indices.shape) < left_out
    pick |= rng.random((n, 1)) < left_out
    indices[pick] = wrong[rng.integers(0, 5, int(pick.sum()))]
    return logits, torch.tensor(indices, device=DEVICE).to(index)


def check(n, experts, chosen, dtype, **how):
    import efgs
    print(f'case balance n={n} experts={experts} chosen={chosen} {dtype} {how}', flush=True)
    logits, indices = inputs(n, experts, chosen, dtype, **how)
    logits.requires_grad_()
    up = torch.tensor(0.37, device=DEVICE)
    loss, counts = efgs.balance_loss(logits, indices)
    z = logits.detach().double().cpu().numpy()
    want, want_counts, gradient = R.balance(z, indices.cpu().numpy(), float(up))
    assert loss.dtype == torch.float32 and counts.dtype == torch.int64 and not counts.requires_grad
    assert np.array_equal(counts.cpu().numpy(), want_counts)
    finite = np.where(np.isfinite(z), z, 0.0)
    spread = (finite.max(1) - finite.min(1)).max(initial=0.0)
    r = (2 * spread + 60) * E
    assert abs(float(loss.detach()) - want) <= (r + (np.ceil(n / 1024) + 40) * E) * abs(want) + 1e-300
    grad = torch.autograd.grad(loss, logits, up)[0]
    assert grad.dtype == logits.dtype
    _, u, least = TYPES[dtype]
    valid = (indices.cpu().numpy() >= 0) & (indices.cpu().numpy() < experts)
    rows = valid.any(1)
    share = want_counts / max(1, want_counts.sum())
    with np.errstate(invalid='ignore', over='ignore'):
        p = np.exp(z - np.where(np.isneginf(z.max(1, keepdims=True)), 0.0, z.max(1, keepdims=True)))
    p = np.where(rows[:, None], p / np.maximum(p.sum(1, keepdims=True), 1e-300), 0.0)
    mean = (p @ share)[:, None]
    factor = float(up) * experts / max(1, rows.sum())
    bar = factor * p * (np.abs(share - mean) * (r + 6 * E) + mean * (r + 45 * E) + share * 2 * E)
    bar += u * (np.abs(gradient) + bar) + least
    off = np.abs(grad.double().cpu().numpy() - gradient)
    assert np.all(off <= bar), (float(np.max(off / np.maximum(bar, 1e-300))), np.unravel_index(np.argmax(off - bar), off.shape))
    assert np.all(grad.cpu().float().numpy()[~rows] == 0)
    return logits, indices, loss, counts, grad


@pytest.mark.parametrize('experts', [1, 2, 3, 4, 8, 9, 16, 31, 32, 60, 64, 65, 128, 250, 256, 257, 512, 1000, 1024, 1025, 2048, 2049, 4096, 5001, 8191, 8192])
@pytest.mark.parametrize('dtype', list(TYPES))
def test_widths(experts, dtype):
    check(203, experts, min(3, experts), dtype, seed=experts)


@pytest.mark.parametrize('n', [1, 2, 3, 4, 15, 16, 17, 64, 255, 256, 257, 5000, 70_001])
@pytest.mark.parametrize('experts,chosen', [(8, 2), (64, 1), (61, 4)])
def test_lengths(n, experts, chosen):
    check(n, experts, chosen, 'f32', seed=n)


@pytest.mark.parametrize('chosen', [0, 1, 2, 7, 64, 65, 300])
def test_choices(chosen):
    check(100, 40, chosen, 'bf16', index=torch.int32)


@pytest.mark.parametrize('left_out', [0.0, 0.7, 1.0])
@pytest.mark.parametrize('experts', [7, 64, 3000])
def test_rows_left_out(left_out, experts):
    _, _, loss, counts, grad = check(150, experts, 2, 'f32', left_out=left_out)
    if left_out == 1.0:
        assert float(loss.detach()) == 0 and int(counts.sum()) == 0 and torch.all(grad == 0)


@pytest.mark.parametrize('experts', [7, 64, 3000])
@pytest.mark.parametrize('dtype', list(TYPES))
def test_masked_logits_and_rows_of_nothing_else(experts, dtype):
    check(100, experts, 2, dtype, masked=0.5)
    import efgs
    logits, indices = inputs(50, experts, 2, dtype)
    logits[4] = -float('inf')
    logits[5] = torch.finfo(TYPES[dtype][0]).min
    logits.requires_grad_()
    loss, _ = efgs.balance_loss(logits, indices)
    want, _, gradient = R.balance(logits.detach().double().cpu().numpy(), indices.cpu().numpy())
    assert abs(float(loss.detach()) - want) <= 1e-5 * want
    grad = torch.autograd.grad(loss, logits)[0]
    assert torch.all(grad[4] == 0) and torch.all(torch.isfinite(grad))


@pytest.mark.parametrize('experts', [7, 64, 3000])
def test_what_stands_in_rows_left_out_reaches_nothing(experts):
    import efgs
    logits, indices = inputs(90, experts, 2, 'f32', left_out=0.3)
    out = ((indices < 0) | (indices >= experts)).all(1)
    assert int(out.sum()) > 5
    results = []
    for value in (0.0, float('nan'), float('inf')):
        z = logits.clone()
        z[out] = value
        z.requires_grad_()
        loss, counts = efgs.balance_loss(z, indices)
        results.append((loss.detach(), counts, torch.autograd.grad(loss, z)[0]))
    for other in results[1:]:
        for a, b in zip(results[0], other):
            assert torch.equal(a, b)
    z = logits.clone()
    z[int((~out).nonzero()[0]), 0] = float('nan')
    assert bool(torch.isnan(efgs.balance_loss(z, indices)[0]))


def test_shapes_and_strides():
    import efgs
    base = torch.randn(12, 5, 7, device=DEVICE)
    indices = torch.randint(0, 12, (7, 5, 3), device=DEVICE)
    z = base.permute(2, 1, 0).requires_grad_()
    a = efgs.balance_loss(z, indices)
    b = efgs.balance_loss(z.detach().contiguous().view(35, 12), indices.view(35, 3))
    assert torch.equal(a[0].detach(), b[0]) and torch.equal(a[1], b[1])
    assert torch.autograd.grad(a[0], z)[0].shape == (7, 5, 12)
    one = efgs.balance_loss(z, indices[..., 0])
    assert torch.equal(one[1], torch.bincount(indices[..., 0].flatten(), minlength=12))
    alone = efgs.balance_loss(torch.randn(12, device=DEVICE), torch.tensor(3, device=DEVICE))
    assert int(alone[1][3]) == 1
    empty = torch.empty(0, 6, device=DEVICE, requires_grad=True)
    loss, counts = efgs.balance_loss(empty, torch.empty(0, 2, dtype=torch.int64, device=DEVICE))
    assert float(loss.detach()) == 0 and int(counts.sum()) == 0 and torch.autograd.grad(loss, empty)[0].shape == (0, 6)
    off = torch.randn(1 + 40 * 64, device=DEVICE).to(torch.bfloat16)
    view, choice = off[1:].view(40, 64), torch.randint(0, 64, (40,), device=DEVICE)
    assert torch.equal(efgs.balance_loss(view, choice)[0], efgs.balance_loss(view.clone(), choice)[0])


def test_the_same_bits_every_time_and_captured():
    import efgs
    logits, indices = inputs(30_000, 64, 2, 'f32')
    logits.requires_grad_()
    def step():
        loss, counts = efgs.balance_loss(logits, indices)
        return loss, counts, torch.autograd.grad(loss, logits)[0]
    first = [t.detach().clone() for t in step()]
    for a, b in zip(first, step()):
        assert torch.equal(a, b)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in range(1, 4):
        other = inputs(30_000, 64, 2, 'f32', seed=seed)
        with torch.no_grad():
            logits.copy_(other[0])
            indices.copy_(other[1])
        graph.replay()
        torch.cuda.synchronize()
        got = [t.detach().clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)


@pytest.mark.parametrize('experts', [3, 8, 300])
def test_even_choices_have_no_gradient(experts):
    """Every expert chosen as often as the others: the loss is 1 and its gradient zero, not what the probabilities' rounded sum leaves."""
    import efgs
    logits = torch.randn(7, experts, generator=torch.Generator(DEVICE).manual_seed(2), device=DEVICE).requires_grad_()
    indices = torch.arange(experts, device=DEVICE).expand(7, experts)
    loss, counts = efgs.balance_loss(logits, indices)
    assert torch.all(counts == 7) and abs(float(loss.detach()) - 1.0) <= 2.0 ** -20
    loss.backward()
    assert torch.all(logits.grad == 0)


@pytest.mark.parametrize('n', [1, 2, 203])
@pytest.mark.parametrize('experts', [4094, 4098, 4100, 4102, 4104, 6146, 8186, 8188, 8190])
@pytest.mark.parametrize('dtype', list(TYPES))
def test_even_widths_of_many_experts(experts, n, dtype):
    """Multiples of two, four and eight up to the largest ones; one row, whose only block makes the loss too, and several."""
    check(n, experts, 3, dtype, seed=experts + n, left_out=0.0 if n == 1 else 0.1)


def test_a_penalty_on_the_gradient_raises():
    """The gradient depends on the logits themselves: what is differentiated through it raises, also where the upstream gradient asks for none."""
    import efgs
    logits, indices = inputs(40, 16, 2, 'f32')
    logits.requires_grad_()
    loss, _ = efgs.balance_loss(logits, indices)
    grad, = torch.autograd.grad(loss, logits, create_graph=True)
    want, = torch.autograd.grad(efgs.balance_loss(logits, indices)[0], logits)
    assert grad.requires_grad and not want.requires_grad and torch.equal(grad, want)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        torch.autograd.grad(loss + grad.pow(2).sum(), logits, retain_graph=True)
    with pytest.raises(RuntimeError, match='once_differentiable'):
        (loss + grad.pow(2).sum()).backward()
