"""The launch shapes that long training has and small tests do not: steps of more than a million elements (two pieces a thread), full
launches of many tensors, decoding of many states, norms of several rounds a block, and 32-bit and 64-bit indices through every form of the
table gradient. Bars as in test_gpu_adamw.py and test_gpu_embedding.py."""
import numpy as np
import pytest
import torch

import training_ref as R
from test_gpu_adamw import DEFAULTS, E, TYPES, _check_parameter, _check_step, _host, _make
from test_gpu_embedding import _check_gradient, _plain

pytestmark = pytest.mark.gpu

DEVICE = 'cuda:0'


@pytest.mark.parametrize('n, dtype', [((1 << 20) + 1, 'f32'), (1_300_003, 'f32'), (1_300_003, 'bf16'), (2_097_152, 'f16')])
@pytest.mark.parametrize('rates', [1, 2, 5, 7])
@pytest.mark.parametrize('max_norm', [None, 0.5])
def test_steps_of_more_than_a_million_elements(n, dtype, rates, max_norm):
    """Two pieces a thread: whole blocks and a tail, one rate and rates by column."""
    import efgs
    print(f'case adamw32 large n={n} {dtype} rates={rates} {max_norm}', flush=True)
    kind, rounding, least = TYPES[dtype]
    p, g = _make(n, kind, kind, rates)
    hyper = dict(DEFAULTS, lr=[1e-3 * (k + 1) for k in range(rates)] if rates > 1 else 1e-3)
    opt = efgs.AdamW([p], max_grad_norm=max_norm, **hyper)
    gradient = _host(g)
    coefficient = R.clip_coefficient([gradient], max_norm)[1] if max_norm else 1.0
    m = v = np.zeros(n)
    for step in (1, 2):
        before = _host(p), m, v
        opt.step()
        state = opt.state[p]
        after = _host(p), _host(state['exp_avg']), _host(state['exp_avg_sq'])
        if max_norm:
            want_p, want_m, want_v = R.adamw(before[0], gradient, m, v, step, hyper['lr'], 0.9, 0.999, hyper['eps'], hyper['weight_decay'], coefficient)
            # (the coefficient: the norm, the sum, the quotient and the product, 4 e of the gradient's terms and 8 e of their squares)
            size = 0.9 * np.abs(m) + 0.1 * np.abs(gradient) * coefficient
            assert np.all(np.abs(after[1] - want_m) <= 10 * E * size + 1e-44) and np.all(np.abs(after[2] - want_v) <= 16 * E * want_v + 1e-44)
            _check_parameter(before[0], after[0], want_p, want_m, want_v, size * 10 / 6, step, hyper, rounding, least)
        else:
            _check_step(before, after, gradient, step, hyper, rounding, least)
        m, v = after[1:]


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('mean', [700, 30_000])
@pytest.mark.parametrize('rates', [1, 3])
def test_full_launches_of_one_group(bits, mean, rates):
    """150 tensors of odd sizes in one group (launches of 72 or 60 tensors, the search past its first 64), bit for bit as single tensors, which
    one piece a thread takes; of 30,000 elements in the mean two pieces take them together. Moments of all at once as one by one."""
    import efgs
    print(f'case adamw full launches {bits} {mean} {rates}', flush=True)
    rng = np.random.default_rng(mean)
    sizes = [1 + 2 * int(rng.integers(0, mean)) for _ in range(150)]
    together, alone = ([_make(n, torch.float32, torch.float32, k)[0] for k, n in enumerate(sizes)] for _ in range(2))
    hyper = dict(DEFAULTS, lr=[1e-3, 2e-3, 3e-3] if rates == 3 else 1e-3, state_bits=bits, seed=5)
    opt = efgs.AdamW(together, **hyper)
    singles = [efgs.AdamW([p], **hyper) for p in alone]
    for _ in range(2):
        opt.step()
        for s in singles:
            s.step()
    moments = opt.moments(together)
    assert len(moments) == 150
    for p, q, s, (m, v) in zip(together, alone, singles, moments):
        assert torch.equal(p, q)
        for key, value in opt.state[p].items():
            other = s.state[q][key]
            assert torch.equal(value, other) if isinstance(value, torch.Tensor) else value == other
        other_m, other_v = s.moments(q)
        assert torch.equal(m, other_m) and torch.equal(v, other_v)


@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
@pytest.mark.parametrize('sizes', [(40_000_003,), (5, 40_000_003, 1, 4097), (17_000_001, 33, 68_000_003)])
def test_norm_of_several_rounds_a_block(dtype, sizes):
    """Whole numbers from 1 to 4 throughout, whose squares' sum 64 bits hold exactly: a piece of 1,024 that is left out or counted twice moves
    the norm by 1e-5 of it at the least. Then threes in a sea of 2^-20 at both ends, at pieces' edges and between: one of them by 3 %."""
    import efgs
    print(f'case norm large {dtype} {sizes}', flush=True)
    generator = torch.Generator(DEVICE).manual_seed(len(sizes))
    tensors = [torch.randint(1, 5, (n + 1,), generator=generator, device=DEVICE).to(TYPES[dtype][0])[1:] for n in sizes]
    want = float(np.sqrt(sum(int((t.long() ** 2).sum()) for t in tensors)))
    assert float(efgs.grad_norm(tensors)) == pytest.approx(want, rel=2 * E)
    for t in tensors:
        t.fill_(2.0 ** -20)
    n = tensors[-1].numel()
    places = sorted({0, 1, 1023, 1024, 8191, 8192, 8193, n // 3, n // 2, n - 1025, n - 4, n - 3, n - 2, n - 1} & set(range(n)))
    for k in places:
        tensors[-1][k] = 3.0
    assert float(efgs.grad_norm(tensors)) == pytest.approx(float(np.sqrt(9.0 * len(places) + sum(t.numel() for t in tensors) * 2.0 ** -40)), rel=4 * E)


@pytest.mark.parametrize('index', [torch.int32, torch.int64])
@pytest.mark.parametrize('n', [5000, 12_000, 30_000, 300_000, 1_100_000])
@pytest.mark.parametrize('rows', [300, 4096, 5000, 70_000])
def test_index_types_through_every_form(index, n, rows):
    """Ranks, the scatter that counts alone, the table with one and with four keys a thread, tiles of one to four: both types, with indices
    outside the table, those of 64 bits past 32 bits too (their low bits name a row)."""
    import efgs
    print(f'case embedding {index} n={n} rows={rows}', flush=True)
    rng = np.random.default_rng(n + rows)
    indices = (rows * rng.random(n) ** 2).astype(np.int64)
    wrong = [-1, rows, rows + 3, -(1 << 31), (1 << 31) - 1]
    if index == torch.int64:
        wrong += [1 << 32, (1 << 32) + 3, (1 << 32) + rows - 1, -(1 << 32), -(1 << 32) + 2, (1 << 63) - 1, -(1 << 63), (1 << 40) + 7]
    pick = rng.random(n) < 0.05
    indices[pick] = np.asarray(wrong)[rng.integers(0, len(wrong), int(pick.sum()))]
    indices = torch.tensor(indices, device=DEVICE).to(index)
    table = torch.randn(rows, 4, device=DEVICE, requires_grad=True)
    out = efgs.embedding(indices, table, 1.5, 2)
    assert torch.equal(out, _plain(indices, table, 1.5))
    grad = torch.randn(n, 4, device=DEVICE)
    out.backward(grad)
    _check_gradient(table.grad, indices, grad, rows, 1.5, 'f32', 2)


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('skipped', [1, 10])
def test_a_step_left_out_counts(bits, skipped):
    """Steps left out for their norm count in t: the first one that is taken corrects its moments, of one gradient, as of step
    `skipped` + 1, and a program that wants another t sets the state's `step`."""
    import efgs
    p, g = _make(700, torch.float32, torch.float32, 3)
    opt = efgs.AdamW([p], state_bits=bits, max_grad_norm=1e9, **DEFAULTS)
    before, kept = _host(p), g.clone()
    g[5] = float('inf')
    for _ in range(skipped):
        opt.step()
    assert opt.state[p]['step'] == skipped and np.array_equal(_host(p), before)
    assert not any(bool(x.any()) for x in opt.moments(p))
    g.copy_(kept)
    opt.step()
    assert opt.state[p]['step'] == skipped + 1
    want = R.adamw(before, _host(g), 0.0, 0.0, skipped + 1, DEFAULTS['lr'], 0.9, 0.999, DEFAULTS['eps'], DEFAULTS['weight_decay'])[0]
    np.testing.assert_allclose(_host(p), want, rtol=8 * E, atol=64 * E * DEFAULTS['lr'])
    q = torch.tensor(before, device=DEVICE).float().requires_grad_()
    q.grad = kept.clone()
    other = efgs.AdamW([q], state_bits=bits, max_grad_norm=1e9, **DEFAULTS)
    q.grad[5] = float('inf')
    other.step()
    if not bool(torch.isfinite(other.grad_norm)):
        other.state[q]['step'] -= 1
    q.grad.copy_(kept)
    other.step()
    want = R.adamw(before, _host(g), 0.0, 0.0, 1, DEFAULTS['lr'], 0.9, 0.999, DEFAULTS['eps'], DEFAULTS['weight_decay'])[0]
    np.testing.assert_allclose(_host(q), want, rtol=8 * E, atol=64 * E * DEFAULTS['lr'])
