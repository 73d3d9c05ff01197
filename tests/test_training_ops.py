"""The training operators without a GPU: refusals of the C entry points and of the Python ones before any device work, and
the arithmetic that the 8-bit AdamW states rest on (bound of the ratio, coding, dither), on the 64-bit oracle."""
import ctypes

import numpy as np
import pytest
import torch

import training_ref as R


def _adamw_call(group=None, n_groups=1, n_tensors=1, grad_norm=None, max_norm=1.0, **tensor):
    from efgs import _lib
    g = _lib.AdamWGroup()
    g.lrs[0], g.beta1, g.beta2, g.eps, g.n_lrs, g.state_bits = 1e-3, 0.9, 0.999, 1e-8, 1, 32
    for k, v in (group or {}).items():
        if k == 'lr':
            g.lrs[0] = v
        else:
            setattr(g, k, v)
    t = _lib.AdamWTensor()
    t.param = t.grad = t.exp_avg = t.exp_avg_sq = t.root_scale = 0x1000   # never dereferenced
    t.n_elements, t.step, t.ratio_bound = 4, 1, 7.0
    for k, v in tensor.items():
        setattr(t, k, v)
    rc = _lib.lib.efgs_adamw_step(ctypes.byref(t), n_tensors, ctypes.byref(g), n_groups, grad_norm, max_norm, 0, None)
    return rc, _lib.lib.efgs_last_error().decode()


@pytest.mark.parametrize('call, word', [
    (dict(n_tensors=-1), 'invalid'),
    (dict(n_groups=-1), 'invalid'),
    (dict(group=dict(n_lrs=0)), 'learning rates'),
    (dict(group=dict(n_lrs=8)), 'learning rates'),
    (dict(group=dict(lr=float('nan'))), 'finite'),
    (dict(group=dict(beta1=1.0)), 'betas'),
    (dict(group=dict(beta2=-0.1)), 'betas'),
    (dict(group=dict(beta2=float('nan'))), 'betas'),
    (dict(group=dict(eps=-1e-8)), 'eps'),
    (dict(group=dict(weight_decay=float('inf'))), 'decay'),
    (dict(group=dict(state_bits=16)), '32 or 8'),
    (dict(group=dict(state_bits=8, beta1=0.99, beta2=0.9)), 'beta1^2'),
    (dict(group=dict(state_bits=8), root_scale=None), 'scales'),
    (dict(group=dict(state_bits=8), ratio_bound=0.0), 'bound'),
    (dict(group=dict(state_bits=8), ratio_bound=float('nan')), 'bound'),
    (dict(group_index=1), 'group'),
    (dict(n_elements=-1), 'count'),
    (dict(n_elements=(1 << 33) + 1), 'count'),
    (dict(step=0), 'counts from 1'),
    (dict(param_type=3), 'type'),
    (dict(grad_type=-1), 'type'),
    (dict(param=None), 'null'),
    (dict(exp_avg_sq=None), 'null'),
    (dict(grad_norm=0x1000, max_norm=0.0), 'positive'),
])
def test_adamw_step_refuses(call, word):
    if 'group_index' in call:
        from efgs import _lib
        g, t = _lib.AdamWGroup(), _lib.AdamWTensor()
        g.lrs[0], g.beta2, g.n_lrs, g.state_bits = 1e-3, 0.9, 1, 32
        t.group, t.step = call['group_index'], 1
        rc, message = _lib.lib.efgs_adamw_step(ctypes.byref(t), 1, ctypes.byref(g), 1, None, 0.0, 0, None), _lib.lib.efgs_last_error().decode()
    else:
        rc, message = _adamw_call(**call)
    assert rc == 1 and word in message, (rc, message)


def test_adamw_step_of_nothing_is_accepted():
    from efgs import _lib
    assert _lib.lib.efgs_adamw_step(None, 0, None, 0, None, 0.0, 0, None) == 0
    assert _adamw_call(n_elements=0, param=None, grad=None)[0] == 0


def test_other_entry_points_refuse():
    from efgs import _lib
    lib, fake = _lib.lib, ctypes.c_void_p(0x1000)
    none = _lib.ALLOC_FN(lambda ctx, n: 0)
    state = _lib.AdamWState()
    state.n_elements = 4
    assert lib.efgs_adamw_moments(ctypes.byref(state), 1, None) == 1
    assert lib.efgs_adamw_moments(None, 1, None) == 1 and lib.efgs_adamw_moments(None, 0, None) == 0
    norm = _lib.NormTensor()
    norm.data, norm.n_elements = 0x1000, 4
    assert lib.efgs_grad_norm(ctypes.byref(norm), 1, None, none, None, None) == 1
    assert lib.efgs_grad_norm(ctypes.byref(norm), 1, fake, none, None, None) == 5    # the allocation fails
    norm.type = 7
    assert lib.efgs_grad_norm(ctypes.byref(norm), 1, fake, none, None, None) == 1
    forward = lambda **k: lib.efgs_embedding_forward(*{**dict(i=fake, b=8, n=4, t=fake, r=3, c=5, s=5, ty=0, sc=1.0, o=fake, st=None), **k}.values())
    assert forward(b=2) == 1 and forward(n=-1) == 1 and forward(c=1 << 31) == 1 and forward(ty=9) == 1 and forward(sc=float('inf')) == 1
    assert forward(i=None) == 1 and forward(t=None) == 1 and forward(o=None) == 1 and forward(s=-1) == 1
    assert forward(n=0, i=None, o=None) == 0 and forward(c=0) == 0
    backward = lambda **k: lib.efgs_embedding_backward(
        *{**dict(i=fake, b=8, n=4, g=fake, r=3, c=5, ty=0, sc=1.0, p=-1, o=fake, a=none, ctx=None, st=None), **k}.values())
    assert backward(g=None) == 1 and backward(o=None) == 1 and backward(sc=float('nan')) == 1 and backward(r=-1) == 1
    assert backward() == 5                                                            # the allocation fails
    assert backward(n=(1 << 31) - 1, r=(1 << 31) - 1) == 1                            # more items than a launch counts
    assert backward(r=0, o=None) == 0


@pytest.mark.parametrize('bad', [dict(betas=(0.9, 1.0)), dict(state_bits=16), dict(betas=(0.95, 0.9), state_bits=8), dict(lr=[1e-3] * 8), dict(lr=[]),
                                 dict(max_grad_norm=0.0), dict(max_grad_norm=float('nan')), dict(eps=-1.0)])
def test_adamw_refuses_values(bad):
    import efgs
    with pytest.raises(ValueError):
        efgs.AdamW([torch.nn.Parameter(torch.zeros(3))], **bad)


def test_python_entry_points_refuse_host_tensors():
    import efgs
    p = torch.nn.Parameter(torch.zeros(3))
    opt = efgs.AdamW([p])
    opt.step()                      # no gradients: nothing to do
    assert opt.grad_norm is None
    p.grad = torch.ones(3)
    with pytest.raises(ValueError, match='GPU'):
        opt.step()
    with pytest.raises(ValueError, match='no state'):
        opt.moments(p)
    with pytest.raises(ValueError, match='GPU'):
        efgs.embedding(torch.zeros(2, dtype=torch.int64), torch.zeros(3, 3))
    with pytest.raises(ValueError, match='two dimensions'):
        efgs.embedding(torch.zeros(2, dtype=torch.int64), torch.zeros(3))
    with pytest.raises(ValueError, match='int32 or int64'):
        efgs.embedding(torch.zeros(2), torch.zeros(3, 3))
    with pytest.raises(ValueError, match='at least one'):
        efgs.grad_norm([])
    with pytest.raises(ValueError, match='GPU'):
        efgs.grad_norm(torch.zeros(3))


@pytest.mark.parametrize('betas', [(0.9, 0.999), (0.9, 0.95), (0.0, 0.9), (0.95, 0.999)])
def test_ratio_bound_is_the_largest_ratio(betas):
    """|m| <= B sqrt(v) over any gradients, and the gradients beta1^k / beta2^k (latest first) come near it."""
    from efgs import _lib
    b1, b2 = betas
    bound = R.ratio_bound(b1, b2)
    assert _lib.lib.efgs_adamw_ratio_bound(b1, b2) == pytest.approx(bound, rel=1e-12)
    rng = np.random.default_rng(3)
    streams = rng.normal(size=(200, 64)) * np.exp(rng.normal(size=(200, 64)) * 3)
    worst = (b1 / b2) ** np.arange(400)[::-1][:, None] if b1 else np.eye(2)[1][:, None]
    reached = 0.0
    for gradients in (streams, worst):
        m = v = np.zeros(gradients.shape[1])
        for g in gradients:
            m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
            assert np.all(np.abs(m) <= bound * np.sqrt(v) * (1 + 1e-12))
        reached = np.max(np.abs(m) / np.sqrt(v))
    assert reached > 0.99 * bound


@pytest.mark.parametrize('kind', [R.ROOT, R.RATIO])
def test_codes_are_monotonic_and_positions_meet_them(kind):
    values = R.code_value(np.arange(kind['codes']), kind)
    assert values[0] == 0.0 and np.all(np.diff(values) > 0) and values[-1] == R.TOP - kind['c']
    np.testing.assert_allclose(R.code_position(values, kind), np.arange(kind['codes']), atol=1e-9)
    middle = (values[1:] + values[:-1]) / 2
    np.testing.assert_allclose(R.code_position(middle, kind), np.arange(kind['codes'] - 1) + 0.5, atol=1e-9)
    # steps: c / 16 up to twice c, then a 16th to a 32nd of y + c
    assert np.all(np.diff(values) / (values[:-1] + kind['c']) <= 1 / 16 + 1e-12)


def test_dither_is_uniform_over_elements_and_over_steps():
    """Means and correlations over 4,096 elements x 256 steps: standard errors 1 / sqrt(12 n) and 1 / sqrt(n), five of them allowed."""
    drawn = [np.stack(x) for x in zip(*(R.dither(4096, t, 11) for t in range(1, 257)))]
    for x in drawn:
        n = x.size
        assert abs(x.mean() - 0.5) < 5 / np.sqrt(12 * n)
        assert np.all(np.abs(x.mean(0) - 0.5) < 5.5 / np.sqrt(12 * 256)) and np.all(np.abs(x.mean(1) - 0.5) < 5 / np.sqrt(12 * 4096))
        y = (x - 0.5) * np.sqrt(12)
        for pair in (y[1:] * y[:-1], y[:, 1:] * y[:, :-1]):
            assert abs(pair.mean()) < 5 / np.sqrt(pair.size)
    both = (drawn[0] - 0.5) * (drawn[1] - 0.5) * 12
    assert abs(both.mean()) < 5 / np.sqrt(both.size)


def test_coding_is_right_in_the_mean_where_nearest_would_stand_still():
    """r that shrinks by 0.05 % a step (beta2 = 0.999, no gradient) follows its course in the mean of 4,096 elements, though a
    code's step is 3 to 6 %. Each element's relative variance is at most (0.0005 * 400 steps) * (1/16) at the last, so
    the mean of 4,096 lies within 5 * sqrt(0.0125 / 4096) = 0.9 % of it."""
    n, bound = 4096, R.ratio_bound(0.9, 0.999)
    rng = np.random.default_rng(0)
    r0 = np.exp(rng.normal(size=n) * 0.5)
    keep = r0.reshape(-1, 256).argmax(1) + np.arange(n // 256) * 256        # each block's maximum stays where it is
    r = r0.copy()
    for t in range(1, 401):
        v = np.where(np.isin(np.arange(n), keep), r0 ** 2, 0.999 * r ** 2)
        _, root, scale, _ = R.encode_positions(np.zeros(n), v, bound)
        low, _ = R.dither(n, t, 5)
        r = R.code_value(np.minimum(np.floor(root + low), 255), R.ROOT) * np.repeat(scale, 256)
    moved = ~np.isin(np.arange(n), keep)
    course = (r / r0)[moved].mean() / 0.999 ** 200
    assert abs(course - 1) < 0.009 + 0.0005, course   # (0.05 %: the maximum's own code is not quite its value)


def test_eight_bit_training_follows_the_moments():
    """300 steps of noisy gradients whose size varies by 10^4 within a block: m / sqrt(v) from 8-bit states stays near the
    64-bit one for large and small elements alike (rms difference under 0.15 of the rms ratio of about 0.23 + mean 0.5)."""
    n, (b1, b2) = 1024, (0.9, 0.999)
    bound, rng = R.ratio_bound(b1, b2), np.random.default_rng(2)
    size = 10.0 ** rng.uniform(-4, 0, n)
    m = v = np.zeros(n)
    ratio, root, scale = np.zeros(n, np.int64), np.zeros(n, np.int64), np.zeros(n // 256)
    for t in range(1, 301):
        g = size * (0.5 + rng.normal(size=n))
        m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        m8, v8, _, _ = R.decode(ratio, root, scale, bound)
        m8, v8 = b1 * m8 + (1 - b1) * g, b2 * v8 + (1 - b2) * g * g
        at_ratio, at_root, scale, negative = R.encode_positions(m8, v8, bound)
        low, high = R.dither(n, t, 9)
        root = np.minimum(np.floor(at_root + low), 255).astype(np.int64)
        ratio = np.minimum(np.floor(at_ratio + high), 127).astype(np.int64) + 128 * negative
    want, got = m / np.sqrt(v), m8 / np.sqrt(v8)
    for part in (size < 1e-3, size > 1e-1):
        assert np.sqrt(np.mean((got - want)[part] ** 2)) < 0.15 * np.sqrt(np.mean(want[part] ** 2)) + 0.05
        assert abs(np.mean((got - want)[part])) < 0.02
        assert abs(np.mean((np.sqrt(v8 / v))[part]) - 1) < 0.03
