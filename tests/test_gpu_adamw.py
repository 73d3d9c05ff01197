"""efgs.AdamW and efgs.grad_norm on the GPU against the 64-bit oracle (oracle/training_ref.py).

Bars, e = 2^-24 the rounding of a float32 operation:
  m, v          three roundings of terms no larger than beta1 |m| + (1 - beta1) |g| (squared ones for v), and the
                rounded constants (1 - beta and beta, a further e each): 6 e of that sum.
  p             the update's own relative error (m over sqrt(v): 3 + 6 + 6 operations and the step size's rounding) of at most
                24 e of |lr / (1 - beta1^t)| (beta1 |m| + (1 - beta1) |g|) / (1 - beta1) ... bounded by 32 e of |update| plus 6 e of
                the sum above through the update's slope; 3 e |p| for the product and the sum; half a step of the
                parameter's type (e, 2^-8 or 2^-11 of |p|) and, float16, half its least step 2^-25.
  codes         a code is floor(position + dither); float32 gives z = y + c to 10 e, a position to 32 * 10 e = 2^-15.6 < 2^-15.
  scales        12 e relative.
  norm          sums in 64 bits, one rounding: 2 e (and the square root's).
"""
import numpy as np
import pytest
import torch

import training_ref as R

pytestmark = pytest.mark.gpu

E = 2.0 ** -24
TYPES = {'f32': (torch.float32, E, 0.0), 'bf16': (torch.bfloat16, 2.0 ** -8, 0.0), 'f16': (torch.float16, 2.0 ** -11, 2.0 ** -25)}
DEVICE = 'cuda:0'
DEFAULTS = dict(lr=3e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.05)


def _host(t):
    return t.detach().double().cpu().numpy().reshape(-1)


def _make(n, dtype, grad_dtype, seed, offset=0, spread=1.5):
    """A parameter (a view `offset` elements into its storage) and its gradient, a tenth of it zeros."""
    rng = np.random.default_rng(seed)
    g = rng.normal(size=n) * np.exp(rng.normal(size=n) * spread - 3) * (rng.random(n) > 0.1)
    storage = torch.zeros(n + offset, dtype=dtype, device=DEVICE)
    storage[offset:] = torch.tensor(rng.normal(size=n), device=DEVICE).to(dtype)
    p = storage[offset:].requires_grad_()
    grads = torch.zeros(n + offset, dtype=grad_dtype, device=DEVICE)
    grads[offset:] = torch.tensor(g, device=DEVICE).to(grad_dtype)
    if grad_dtype == dtype:
        p.grad = grads[offset:]
        return p, p.grad
    p.grad = None
    return p, grads[offset:]


def _check_step(before, after, g, step, hyper, rounding, least, coefficient=1.0):
    """after = (p, m, v) read back against the oracle's step from before."""
    (p0, m0, v0), (p1, m1, v1) = before, after
    b1, b2 = hyper['betas']
    want_p, want_m, want_v = R.adamw(p0, g, m0, v0, step, hyper['lr'], b1, b2, hyper['eps'], hyper['weight_decay'], coefficient)
    size_m = b1 * np.abs(m0) + (1 - b1) * np.abs(g) * coefficient
    assert np.all(np.abs(m1 - want_m) <= 6 * E * size_m + 1e-44), np.max(np.abs(m1 - want_m) / (size_m + 1e-300))
    assert np.all(np.abs(v1 - want_v) <= 8 * E * want_v + 1e-44)
    _check_parameter(p0, p1, want_p, want_m, want_v, size_m, step, hyper, rounding, least)


def _check_parameter(p0, p1, want_p, want_m, want_v, size_m, step, hyper, rounding, least):
    b1, b2 = hyper['betas']
    lr = np.resize(np.asarray(hyper['lr'], np.float64), len(p0)) if np.ndim(hyper['lr']) else hyper['lr']
    slope = np.abs(lr) / (1 - b1 ** step) / (np.sqrt(want_v / (1 - b2 ** step)) + hyper['eps'])
    bound = slope * (32 * E * np.abs(want_m) + 6 * E * size_m) + 4 * E * np.abs(p0) + (rounding * np.abs(want_p) * (1 + 1e-6) + least)
    off = np.abs(p1 - want_p)
    assert np.all(off <= bound + 1e-44), (np.max(off / (bound + 1e-300)), int(np.argmax(off / (bound + 1e-300))))


@pytest.mark.parametrize('n', [1, 2, 3, 4, 5, 63, 255, 256, 257, 1023, 1024, 1025, 4099, 70_001])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_steps_of_32_bit_states(n, dtype):
    import efgs
    print(f'case adamw32 n={n} {dtype}', flush=True)
    kind, rounding, least = TYPES[dtype]
    p, g = _make(n, kind, kind, n)
    opt = efgs.AdamW([p], **DEFAULTS)
    m = v = np.zeros(n)
    for step in (1, 2, 3):
        before = _host(p), m, v
        opt.step()
        state = opt.state[p]
        after = _host(p), _host(state['exp_avg']), _host(state['exp_avg_sq'])
        assert state['step'] == step
        _check_step(before, after, _host(g), step, DEFAULTS, rounding, least)
        m, v = after[1:]


@pytest.mark.parametrize('offset', [1, 2, 3, 5])
@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_results_do_not_depend_on_alignment(offset, bits, dtype):
    """Views that begin anywhere in their storage, states too, give the aligned tensors' results bit for bit."""
    import efgs
    print(f'case adamw alignment offset={offset} bits={bits} {dtype}', flush=True)
    n, kind = 1543, TYPES[dtype][0]
    results = []
    for at in (0, offset):
        p, _ = _make(n, kind, kind, 7, at)
        opt = efgs.AdamW([p], state_bits=bits, **DEFAULTS)
        opt.step()
        for key, value in opt.state[p].items():
            if isinstance(value, torch.Tensor):
                moved = torch.zeros(value.numel() + at, dtype=value.dtype, device=DEVICE)
                moved[at:] = value
                opt.state[p][key] = moved[at:]
        opt.step()
        results.append([p.detach()] + [x for x in opt.state[p].values() if isinstance(x, torch.Tensor)])
    for a, b in zip(*results):
        assert torch.equal(a, b)


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
@pytest.mark.parametrize('grad', ['f32', 'bf16', 'f16'])
def test_types_of_parameters_and_gradients(bits, dtype, grad):
    """Every pair through the C entry point (torch gives a parameter gradients of its own type)."""
    import ctypes
    from efgs import _lib
    print(f'case adamw types {bits} {dtype} {grad}', flush=True)
    n = 1301
    p, g = _make(n, TYPES[dtype][0], TYPES[grad][0], 5)
    rng = np.random.default_rng(1)
    r = np.exp(rng.normal(size=n) - 4)
    m0, v0 = (r * rng.normal(size=n) * 0.3).astype(np.float32).astype(np.float64), (r * r).astype(np.float32).astype(np.float64)
    group = _lib.AdamWGroup()
    group.lrs[0], group.n_lrs, group.state_bits = DEFAULTS['lr'], 1, bits
    group.beta1, group.beta2, group.eps, group.weight_decay = 0.9, 0.999, DEFAULTS['eps'], DEFAULTS['weight_decay']
    bound = R.ratio_bound(0.9, 0.999)
    ids = dict(f32=0, bf16=1, f16=2)
    t = _lib.AdamWTensor()
    t.param, t.grad, t.param_type, t.grad_type = p.data_ptr(), g.data_ptr(), ids[dtype], ids[grad]
    t.n_elements, t.step, t.ratio_bound = n, 4, bound
    if bits == 32:
        states = [torch.tensor(x, dtype=torch.float32, device=DEVICE) for x in (m0, v0)]
    else:
        ratio, root, scale, negative = R.encode_positions(m0, v0, bound)
        codes = np.minimum(np.round(ratio), 127).astype(np.uint8) + 128 * negative.astype(np.uint8), np.minimum(np.round(root), 255).astype(np.uint8)
        states = [torch.tensor(c, device=DEVICE) for c in codes] + [torch.tensor(scale, dtype=torch.float32, device=DEVICE)]
        m0, v0, _, _ = R.decode(codes[0], codes[1], _host(states[2]), bound)
        t.root_scale = states[2].data_ptr()
    t.exp_avg, t.exp_avg_sq = states[0].data_ptr(), states[1].data_ptr()
    before = _host(p), m0, v0
    _lib.check(_lib.lib.efgs_adamw_step(ctypes.byref(t), 1, ctypes.byref(group), 1, None, 0.0, 3, torch.cuda.current_stream().cuda_stream))
    torch.cuda.synchronize()
    rounding, least = TYPES[dtype][1:]
    if bits == 32:
        _check_step(before, (_host(p), _host(states[0]), _host(states[1])), _host(g), 4, DEFAULTS, rounding, least)
    else:
        _check_coded(before, _host(p), [x.cpu().numpy() for x in states], _host(g), 4, 3, DEFAULTS, rounding, least)


def _check_coded(before, p1, states, g, step, seed, hyper, rounding, least):
    p0, m0, v0 = before
    b1, b2 = hyper['betas']
    bound = R.ratio_bound(b1, b2)
    want_p, m, v = R.adamw(p0, g, m0, v0, step, hyper['lr'], b1, b2, hyper['eps'], hyper['weight_decay'])
    # (decoding the old state is three roundings for u, two for r: a further 8 e of the terms)
    size_m = (b1 * np.abs(m0) + (1 - b1) * np.abs(g)) * 3
    _check_parameter(p0, p1, want_p, m, v, size_m, step, hyper, rounding, least)
    ratio, root, scale, negative = R.encode_positions(m, v, bound)
    np.testing.assert_allclose(states[2], scale, rtol=12 * E)
    low, high = R.dither(len(p0), step, seed)
    # where m's terms cancel, u's error is e of the terms and not of u: a position moves at most 16 a c-step (c / 16) of y
    cancel = 32 * 6 * E * size_m / np.maximum(np.sqrt(v), 1e-300) / bound / (R.RATIO['c'])
    for codes, position, d, top, slack in ((states[0] & 127, ratio, high, 127, cancel), (states[1], root, low, 255, 0.0)):
        value = position + d
        assert np.all((codes >= np.minimum(np.floor(value - 2.0 ** -15 - slack), top)) & (codes <= np.minimum(np.floor(value + 2.0 ** -15 + slack), top)))
    sure = np.abs(m) > 6 * E * size_m
    assert np.array_equal((states[0] >= 128)[sure], negative[sure])


@pytest.mark.parametrize('n', [1, 2, 3, 5, 255, 256, 257, 511, 1021, 1025, 4099, 70_001])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_steps_of_8_bit_states(n, dtype):
    import efgs
    print(f'case adamw8 n={n} {dtype}', flush=True)
    kind, rounding, least = TYPES[dtype]
    p, g = _make(n, kind, kind, n)
    opt = efgs.AdamW([p], state_bits=8, seed=13, **DEFAULTS)
    bound = R.ratio_bound(0.9, 0.999)
    m = v = np.zeros(n)
    for step in (1, 2, 3, 4):
        before = _host(p), m, v
        opt.step()
        s = opt.state[p]
        states = [s[k].cpu().numpy() for k in ('exp_avg_ratio', 'exp_avg_sq_root', 'root_scale')]
        assert s['step'] == step and s['ratio_bound'] == bound and states[2].shape == ((n + 255) // 256,)
        _check_coded(before, _host(p), states, _host(g), step, 13, DEFAULTS, rounding, least)
        m, v, _, _ = R.decode(*states, bound)
        got_m, got_v = opt.moments(p)
        np.testing.assert_allclose(_host(got_m), m, rtol=6 * E, atol=1e-44)
        np.testing.assert_allclose(_host(got_v), v, rtol=6 * E, atol=1e-44)


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('columns', [2, 3, 5, 7])
def test_learning_rates_by_column(bits, columns):
    import efgs
    print(f'case adamw rates {bits} {columns}', flush=True)
    rows = 1237
    p, g = _make(rows * columns, torch.float32, torch.float32, columns)
    hyper = dict(DEFAULTS, lr=[1e-3 * (k + 1) for k in range(columns)])
    opt = efgs.AdamW([p], state_bits=bits, **hyper)
    before = _host(p), np.zeros(rows * columns), np.zeros(rows * columns)
    opt.step()
    want, m, v = R.adamw(before[0], _host(g), 0.0, 0.0, 1, hyper['lr'], 0.9, 0.999, hyper['eps'], hyper['weight_decay'])
    _check_parameter(before[0], _host(p), want, m, v, 0.1 * np.abs(_host(g)), 1, hyper, E, 0.0)


def _many(count, bits_of, seed):
    rng = np.random.default_rng(seed)
    groups = []
    for k in range(count):
        p, _ = _make(int(rng.integers(1, 3000)), *[TYPES[('f32', 'bf16', 'f16')[k % 3]][0]] * 2, seed * 1000 + k)
        groups.append(dict(params=[p], lr=1e-3 * (1 + k % 11), weight_decay=0.01 * (k % 4), betas=(0.9, 0.99 + 0.001 * (k % 5)), state_bits=bits_of(k)))
    return groups


@pytest.mark.parametrize('count', [2, 41, 130])
def test_many_tensors_give_the_results_of_single_ones(count):
    """More tensors than a launch takes, each in a group of its own (more groups than a launch takes), 8-bit and 32-bit states
    together, bit for bit as if each had an optimizer of its own."""
    import efgs
    print(f'case adamw many {count}', flush=True)
    together = _many(count, lambda k: 8 if k % 2 else 32, count)
    alone = _many(count, lambda k: 8 if k % 2 else 32, count)
    opt = efgs.AdamW(together, seed=3)
    singles = [efgs.AdamW([g], seed=3) for g in alone]
    for _ in range(2):
        opt.step()
        for s in singles:
            s.step()
    for g, h, s in zip(together, alone, singles):
        p, q = g['params'][0], h['params'][0]
        assert torch.equal(p, q)
        for key, value in opt.state[p].items():
            other = s.state[q][key]
            assert torch.equal(value, other) if isinstance(value, torch.Tensor) else value == other


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('max_norm', [1e-3, 1e6])
def test_clipping(bits, max_norm):
    import efgs
    print(f'case adamw clip {bits} {max_norm}', flush=True)
    made = [_make(n, torch.float32, torch.float32, n) for n in (5, 4097, 20_001)]
    opt = efgs.AdamW([p for p, _ in made], state_bits=bits, max_grad_norm=max_norm, **DEFAULTS)
    before = [_host(p) for p, _ in made]
    norm, coefficient = R.clip_coefficient([_host(g) for _, g in made], max_norm)
    opt.step()
    assert float(opt.grad_norm) == pytest.approx(norm, rel=4 * E)
    assert (coefficient < 1) == (max_norm < 1)
    for (p, g), p0 in zip(made, before):
        want, m, v = R.adamw(p0, _host(g), 0.0, 0.0, 1, DEFAULTS['lr'], 0.9, 0.999, DEFAULTS['eps'], DEFAULTS['weight_decay'], coefficient)
        # (the coefficient: the norm's rounding, the sum's, the quotient's and the product's, 4 e)
        _check_parameter(p0, _host(p), want, m, v, 2 * 0.1 * np.abs(_host(g)) * coefficient, 1, DEFAULTS, E, 0.0)
        assert torch.equal(g, p.grad)


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('value', [float('inf'), float('nan')])
def test_a_norm_that_is_not_finite_leaves_everything(bits, value):
    import efgs
    made = [_make(n, torch.float32, torch.float32, n) for n in (300, 5000)]
    opt = efgs.AdamW([p for p, _ in made], state_bits=bits, max_grad_norm=1.0, **DEFAULTS)
    opt.step()
    kept = [[p.detach().clone()] + [x.clone() for x in opt.state[p].values() if isinstance(x, torch.Tensor)] for p, _ in made]
    made[1][1][77] = value
    opt.step()
    assert not np.isfinite(float(opt.grad_norm))
    for (p, _), old in zip(made, kept):
        now = [p.detach()] + [x for x in opt.state[p].values() if isinstance(x, torch.Tensor)]
        assert all(torch.equal(a, b) for a, b in zip(now, old))


@pytest.mark.parametrize('value', [float('inf'), float('-inf'), float('nan'), 1e25, -1e25])
def test_an_odd_gradient_stays_in_its_element(value):
    """Without clipping: the element gets what the formula gives (no number, or for a square that overflows an update of zero)
    and, with 8 bits, a zero state; the other elements of its block are as if its gradient were zero."""
    import efgs
    for bits in (32, 8):
        print(f'case adamw odd {value} {bits}', flush=True)
        results = []
        for odd in (True, False):
            p, g = _make(700, torch.float32, torch.float32, 4)
            opt = efgs.AdamW([p], state_bits=bits, **DEFAULTS)
            opt.step()
            p0 = p.detach().clone()
            g[301] = value if odd else 0.0
            opt.step()
            results.append((p.detach().clone(), p0, [x.clone() for x in opt.moments(p)]))
        (p, p0, moments), (q, _, others) = results
        rest = torch.arange(700, device=DEVICE) != 301
        assert torch.equal(p[rest], q[rest])
        assert bool(torch.isfinite(p[rest]).all())
        if abs(value) < float('inf'):
            assert float(p[301]) == pytest.approx(float(p0[301]) * (1 - DEFAULTS['lr'] * DEFAULTS['weight_decay']), rel=3 * E)
        else:
            assert not bool(torch.isfinite(p[301]))
        if bits == 8:
            assert float(moments[0][301]) == 0.0 and float(moments[1][301]) == 0.0
            # (the block's maximum may have been this element's: codes are of another scale then, moments are not far)
            for a, b in zip(moments, others):
                assert torch.allclose(a[rest], b[rest], rtol=0.15, atol=1e-5)


def test_zero_gradients_and_tiny_ones():
    """No gradient from the first step on leaves p to its decay; gradients whose squares are no floats end as zero
    states, and those near the least scale as zero blocks: no code or scale that is not a number."""
    import efgs
    for size in (0.0, 1e-30, 1e-23, 1e-20):
        for bits in (32, 8):
            print(f'case adamw tiny {size} {bits}', flush=True)
            p, g = _make(1000, torch.float32, torch.float32, 9)
            p0 = _host(p)
            g.copy_(torch.sign(g) * size)
            opt = efgs.AdamW([p], state_bits=bits, **DEFAULTS)
            for _ in range(3):
                opt.step()
            moments = opt.moments(p)
            assert all(bool(torch.isfinite(x).all()) for x in moments + (p,))
            # |update| <= lr B (every step), and without gradients nothing but the decay
            allowed = 3 * DEFAULTS['lr'] * 7.3 if size else 0.0
            decay = (1 - DEFAULTS['lr'] * DEFAULTS['weight_decay']) ** 3
            assert np.all(np.abs(_host(p) - p0 * decay) <= allowed + 4 * 3 * E * np.abs(p0))


def test_missing_and_strided_gradients():
    import efgs
    a, b = (torch.randn(33, 17, device=DEVICE, requires_grad=True) for _ in range(2))
    opt = efgs.AdamW([a, b], **DEFAULTS)
    g = torch.randn(17, 33, device=DEVICE)
    a.grad = g.T
    kept, before = b.detach().clone(), _host(a)
    opt.step()
    assert torch.equal(b, kept) and b not in opt.state
    want, m, v = R.adamw(before, _host(g.T.contiguous()), 0.0, 0.0, 1, DEFAULTS['lr'], 0.9, 0.999, DEFAULTS['eps'], DEFAULTS['weight_decay'])
    _check_parameter(before, _host(a), want, m, v, 0.1 * np.abs(_host(g.T.contiguous())), 1, DEFAULTS, E, 0.0)


def test_refusals_on_the_device():
    import efgs
    p = torch.zeros(4, 6, device=DEVICE).T.requires_grad_()
    p.grad = torch.zeros(6, 4, device=DEVICE)
    with pytest.raises(ValueError, match='contiguous'):
        efgs.AdamW([p]).step()
    q = torch.zeros(4, device=DEVICE, dtype=torch.float64, requires_grad=True)
    q.grad = torch.zeros_like(q)
    with pytest.raises(ValueError, match='float32, bfloat16 or float16'):
        efgs.AdamW([q]).step()
    s = torch.zeros(4, device=DEVICE, requires_grad=True)
    s.grad = torch.zeros(4, device=DEVICE).to_sparse()
    with pytest.raises(ValueError, match='dense'):
        efgs.AdamW([s]).step()
    s.grad = torch.ones(4, device=DEVICE)
    opt = efgs.AdamW([s])
    opt.step()
    opt.param_groups[0]['state_bits'] = 8
    with pytest.raises(ValueError, match='exp_avg_ratio'):
        opt.step()
    opt.param_groups[0]['state_bits'] = 32
    opt.state[s]['exp_avg'] = opt.state[s]['exp_avg'].half()
    with pytest.raises(ValueError, match='exp_avg'):
        opt.step()
    assert opt.state[s]['step'] == 1


def test_capture_is_refused():
    import efgs
    p, _ = _make(64, torch.float32, torch.float32, 1)
    opt = efgs.AdamW([p])
    opt.step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match='captured'):
        with torch.cuda.graph(graph):
            opt.step()
    assert opt.state[p]['step'] == 1


def test_on_a_stream_of_its_own():
    """Gradients made and the step taken on a side stream, behind work that keeps it busy."""
    import efgs
    results = []
    for side in (False, True):
        stream = torch.cuda.Stream() if side else torch.cuda.current_stream()
        stream.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(stream):
            p, g = _make(50_000, torch.float32, torch.float32, 2)
            x = torch.ones(2048, 2048, device=DEVICE)
            for _ in range(8):
                x = x @ x * 1e-4
            g.add_(x[0, 0] * 0)
            opt = efgs.AdamW([p], state_bits=8, max_grad_norm=0.5)
            opt.step()
        torch.cuda.current_stream().wait_stream(stream)
        results.append((p.detach().clone(), opt.state[p]['exp_avg_ratio'].clone()))
    assert all(torch.equal(a, b) for a, b in zip(*results))


@pytest.mark.parametrize('bits', [32, 8])
@pytest.mark.parametrize('dtype', ['f32', 'bf16'])
def test_state_dict_round_trip(bits, dtype):
    """A loaded optimizer goes on bit for bit, its states of their own types (a bfloat16 parameter's included)."""
    import copy
    import efgs
    kind = TYPES[dtype][0]
    p, g = _make(1500, kind, kind, 6)
    opt = efgs.AdamW([p], state_bits=bits, **DEFAULTS)
    opt.step()
    q = p.detach().clone().requires_grad_()
    q.grad = g.clone()
    other = efgs.AdamW([q], state_bits=bits, **DEFAULTS)
    other.load_state_dict(copy.deepcopy(opt.state_dict()))
    assert other.state[q]['step'] == 1
    opt.step()
    other.step()
    assert torch.equal(p, q)
    for key, value in opt.state[p].items():
        if isinstance(value, torch.Tensor):
            assert other.state[q][key].dtype == value.dtype and torch.equal(other.state[q][key], value)


def test_states_of_torch_adamw_are_taken_over():
    import efgs
    p, g = _make(999, torch.float32, torch.float32, 8)
    q = p.detach().clone().requires_grad_()
    q.grad = g.clone()
    theirs = torch.optim.AdamW([q], lr=DEFAULTS['lr'], weight_decay=DEFAULTS['weight_decay'])
    theirs.step()
    ours = efgs.AdamW([p], **DEFAULTS)
    ours.load_state_dict({'state': theirs.state_dict()['state'], 'param_groups': ours.state_dict()['param_groups']})
    with torch.no_grad():
        p.copy_(q)
    theirs.step()
    ours.step()
    assert ours.state[p]['step'] == 2
    torch.testing.assert_close(p.detach(), q.detach(), rtol=1e-6, atol=1e-6)


def test_changed_betas_keep_the_coded_moments():
    """8-bit ratios are coded against the bound of the betas of the step that wrote them; a step with other betas reads them by it."""
    import efgs
    p, g = _make(800, torch.float32, torch.float32, 3)
    opt = efgs.AdamW([p], state_bits=8, **DEFAULTS)
    for _ in range(3):
        opt.step()
    m, v = (_host(x) for x in opt.moments(p))
    p0 = _host(p)
    hyper = dict(DEFAULTS, betas=(0.8, 0.95))
    opt.param_groups[0]['betas'] = hyper['betas']
    opt.step()
    want, m1, v1 = R.adamw(p0, _host(g), m, v, 4, hyper['lr'], 0.8, 0.95, hyper['eps'], hyper['weight_decay'])
    _check_parameter(p0, _host(p), want, m1, v1, 3 * (0.8 * np.abs(m) + 0.2 * np.abs(_host(g))), 4, hyper, E, 0.0)
    assert opt.state[p]['ratio_bound'] == R.ratio_bound(0.8, 0.95)


@pytest.mark.parametrize('betas', [(0.8, 0.95), (0.5, 0.9999)])
@pytest.mark.parametrize('n', [3, 800, 4099])
def test_changed_betas_and_a_norm_that_is_not_finite(betas, n):
    """A step that leaves everything keeps the moments also where its group's betas, and with them the bound of the ratios, are
    not those of the state: m to one step of its code (at most a 16th of the coded value and its offset), up to the new bound."""
    import efgs
    p, g = _make(n, torch.float32, torch.float32, 3)
    opt = efgs.AdamW([p], state_bits=8, max_grad_norm=1.0, **DEFAULTS)
    for _ in range(3):
        opt.step()
    m, v = (_host(x) for x in opt.moments(p))
    kept = [p.detach().clone(), opt.state[p]['exp_avg_sq_root'].clone(), opt.state[p]['root_scale'].clone()]
    g[0] = float('inf')
    opt.param_groups[0]['betas'] = betas
    opt.step()
    assert all(torch.equal(a, b) for a, b in zip([p.detach(), opt.state[p]['exp_avg_sq_root'], opt.state[p]['root_scale']], kept))
    bound, top, c = R.ratio_bound(*betas), R.TOP - R.RATIO['c'], R.RATIO['c']
    unit = np.sqrt(v) * bound / top
    y = np.minimum(np.abs(m) / np.where(unit > 0, unit, 1.0), top)
    got, got_v = (_host(x) for x in opt.moments(p))
    assert np.array_equal(got_v, v)
    assert np.all(np.abs(got - np.sign(m) * y * unit) <= ((y + c) / 16 + 1e-5) * unit)


def test_a_step_counts_as_a_change_in_place():
    import efgs
    p, _ = _make(64, torch.float32, torch.float32, 1)
    loss = (p * p).sum()
    efgs.AdamW([p]).step()
    with pytest.raises(RuntimeError, match='modified by an inplace operation'):
        loss.backward()


def test_results_repeat_and_depend_on_the_seed():
    import efgs
    results = []
    for seed in (1, 1, 2):
        p, _ = _make(5000, torch.float32, torch.float32, 5)
        opt = efgs.AdamW([p], state_bits=8, seed=seed, max_grad_norm=1.0)
        for _ in range(3):
            opt.step()
        results.append((p.detach().clone(), opt.state[p]['exp_avg_sq_root'].clone()))
    assert all(torch.equal(a, b) for a, b in zip(results[0], results[1]))
    assert not torch.equal(results[0][1], results[2][1])


def test_training_with_8_bit_states_reaches_what_32_bits_reach():
    """A regression with noisy gradients, 400 steps: the loss with 8-bit states within 10 % of that with 32-bit ones."""
    import efgs
    torch.manual_seed(0)
    x = torch.randn(4096, 64, device=DEVICE) * torch.logspace(-2, 0, 64, device=DEVICE)
    truth = torch.randn(64, 32, device=DEVICE)
    y = x @ truth + 0.1 * torch.randn(4096, 32, device=DEVICE)
    losses = []
    for bits in (32, 8):
        torch.manual_seed(1)
        w = torch.zeros(64, 32, device=DEVICE, requires_grad=True)
        opt = efgs.AdamW([w], lr=2e-2, weight_decay=0.0, state_bits=bits)
        for _ in range(400):
            pick = torch.randint(0, 4096, (256,), device=DEVICE)
            opt.zero_grad()
            ((x[pick] @ w - y[pick]) ** 2).mean().backward()
            opt.step()
        losses.append(float(((x @ w.detach() - y) ** 2).mean()))
    print('losses', losses, flush=True)
    assert losses[1] < 1.1 * losses[0]


def test_a_tensor_past_2_to_the_32_elements():
    """8-bit states and float16 values of 2^32 + 300 elements (26 GB): the last blocks against a small tensor's, whose dithers are
    those of the same indices modulo 2^32."""
    import efgs
    n = (1 << 32) + 300
    print('case adamw past 2^32', flush=True)
    p = torch.zeros(n, dtype=torch.float16, device=DEVICE)
    g = torch.zeros(n, dtype=torch.float16, device=DEVICE)
    tail = torch.randn(300, device=DEVICE).half()
    p[-300:], g[-300:] = tail, tail * 0.5
    p.requires_grad_()
    p.grad = g
    q = tail.clone().requires_grad_()
    q.grad = tail * 0.5
    big, small = efgs.AdamW([p], state_bits=8), efgs.AdamW([q], state_bits=8)
    for _ in range(2):
        big.step()
        small.step()
    torch.cuda.synchronize()
    assert torch.equal(p.detach()[-300:], q.detach())
    for key in ('exp_avg_ratio', 'exp_avg_sq_root'):
        assert torch.equal(big.state[p][key][-300:], small.state[q][key])
    assert torch.equal(big.state[p]['root_scale'][-2:], small.state[q]['root_scale'])
    assert float(efgs.grad_norm([g])) == pytest.approx(float(tail.double().mul(0.5).half().double().norm()), rel=4 * E)


@pytest.mark.parametrize('sizes', [(1,), (4095, 4096, 4097), (1, 0, 7), tuple(range(1, 140)), (3_000_001, 5)])
@pytest.mark.parametrize('dtype', ['f32', 'bf16', 'f16'])
def test_grad_norm(sizes, dtype):
    import efgs
    print(f'case norm {len(sizes)} {dtype}', flush=True)
    kind = TYPES[dtype][0]
    tensors = [torch.randn(n + 1, device=DEVICE).to(kind)[1:] * (k + 1) for k, n in enumerate(sizes)]
    norm = efgs.grad_norm(tensors)
    want = np.sqrt(sum(float((_host(t) ** 2).sum()) for t in tensors))
    assert norm.shape == () and norm.dtype == torch.float32 and float(norm) == pytest.approx(want, rel=4 * E)
    assert torch.equal(norm, efgs.grad_norm(tensors))


def test_grad_norm_of_large_tiny_and_odd_values():
    import efgs
    huge = torch.full((1000,), 1e30, device=DEVICE)
    assert float(efgs.grad_norm([huge])) == pytest.approx(1e30 * np.sqrt(1000), rel=1e-6)
    assert float(efgs.grad_norm([huge * 1e-60 * 1e-9])) == pytest.approx(0.0, abs=1e-37)
    assert float(efgs.grad_norm([torch.full((900,), 1e-35, device=DEVICE)])) == pytest.approx(3e-34, rel=1e-6)
    assert float(efgs.grad_norm([torch.zeros(0, device=DEVICE)])) == 0.0
    assert np.isnan(float(efgs.grad_norm([torch.tensor([1.0, float('nan')], device=DEVICE)])))
    assert float(efgs.grad_norm([torch.tensor([1.0, float('-inf')], device=DEVICE)])) == float('inf')
    strided = torch.randn(40, 50, device=DEVICE).T
    assert float(efgs.grad_norm(strided)) == pytest.approx(float(np.linalg.norm(_host(strided))), rel=4 * E)
